"""``cached_attention`` at the ends of the scales that it takes, for few query rows and for many."""
import pytest
import torch

from atomic_ai_hybrid_b200 import ops
from _cache import BF, attention_inputs, check_attention

pytestmark = pytest.mark.gpu
dev = "cuda"
HALF = 2.0 ** -8  # half a step of bf16

# few query rows a key head, many, many with a prefix, both kinds in one call
SHAPES = [([1, 3], [200, 70], None), ([200], [0], None), ([9, 130], [100, 3], None), ([40, 1], [0, 30], ([90], [0, 0])),
          ([1] * 12, [5] * 12, ([300], [0] * 12))]


@pytest.mark.parametrize("lens,had,prefix", SHAPES)
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-45, -1e-40, 1e-30])
def test_scales_without_weight(lens, had, prefix, scale):
    """Scores that are all (next to) zero: the mean of what a token sees, and no NaN from a masked place times zero."""
    a = attention_inputs(lens, had, 4, 2, 64, BF, dev, prefix=prefix, tracked=True)
    y, _ = check_attention(ops.cached_attention, {**a, "sm_scale": scale}, HALF)
    assert y.isfinite().all()
