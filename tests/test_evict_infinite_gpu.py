"""The kernel's order of infinite masses, as the plain form's."""
import pytest
import torch

from atomic_ai_hybrid_b200 import ops
from _cache import evict_truth
from test_evict_infinite_cpu import evict_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep,recent", [(1, 0), (2, 0), (3, 0), (3, 1), (9, 0), (8, 8)])
def test_infinite_masses(keep, recent):
    args, n, seen = evict_case("cuda")
    want = evict_truth(*args, n, seen, keep, recent)
    ops.cache_evict(*args, n, seen, keep, recent=recent)
    for a, b in zip(args, want):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
