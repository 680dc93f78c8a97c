"""``cached_attention`` at the ends of the scales that it takes, for few query rows and for many."""
import pytest
import torch

from atomic_ai_hybrid_b200 import ops
from _cache import BF, attention_inputs, attention_truth, check_attention, copied, gen

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


def _whole_numbers(lens, had, prefix, seed=0):
    """Queries and keys of small whole numbers: every score is one too, and exact in whatever order it is summed."""
    a = attention_inputs(lens, had, 4, 2, 64, BF, dev, prefix=prefix, tracked=True, seed=seed, behind=0.0)
    g = gen(seed, dev)
    whole = lambda t: torch.randint(-3, 4, t.shape, generator=g, device=dev).to(BF)  # noqa: E731
    return {**a, **{n: whole(a[n]) for n in ("q", "k", "k_cache")}, "cos": None, "sin": None}


@pytest.mark.parametrize("lens,had,prefix", SHAPES)
@pytest.mark.parametrize("scale", [1e4, 3e6, 1e9, -1e12, 1e28])
def test_large_scales(lens, had, prefix, scale):
    """Weights are one over the number of rows that have the largest score: values are weighed by bf16 numbers of at most half a step off
    (2^-8), summed in 32 bits, and rounded once."""
    a = {**_whole_numbers(lens, had, prefix), "sm_scale": scale}
    o = attention_truth(**copied(a))[0]
    y = ops.cached_attention(**copied(a)).double()
    assert y.isfinite().all()
    assert ((y - o).abs() <= 2 * HALF * (o.abs() + 1e-3)).all(), float((y - o).abs().max())


@pytest.mark.parametrize("scale", [1e6, 1e9, 1e12])
def test_large_scales_of_any_scores(scale):
    """The largest score takes all: next to no two of a row's are within 32 bits of one another."""
    for lens, had, prefix in SHAPES:
        a = attention_inputs(lens, had, 4, 2, 64, BF, dev, prefix=prefix)
        check_attention(ops.cached_attention, {**a, "cos": None, "sin": None, "sm_scale": scale}, HALF)


@pytest.mark.parametrize("lens,had,prefix", SHAPES)
@pytest.mark.parametrize("scale", [0.125, 1e4, 3e6, 1e9, -1e12, 1e28])
def test_masses_at_large_scales(lens, had, prefix, scale):
    """Exact scores, so masses are whole shares, counted in 32 bits."""
    a = {**_whole_numbers(lens, had, prefix), "sm_scale": scale}
    _, _, _, mass, held, _ = attention_truth(**copied(a))
    b = copied(a)
    ops.cached_attention(**b)
    live = a["slots"].long()
    err = (b["mass"].double() - mass)[live].abs()
    assert (err <= 1e-5 * (1 + mass[live].abs())).all(), float(err.max())
    assert torch.equal(b["held"], held)


@pytest.mark.parametrize("scale", [1e6, 1e9, 1e12])
def test_masses_of_any_large_scores_stay_in_bounds(scale):
    for lens, had, prefix in SHAPES:
        a = attention_inputs(lens, had, 4, 2, 64, BF, dev, prefix=prefix, tracked=True)
        before = a["mass"].clone()
        ops.cached_attention(**{**a, "sm_scale": scale})
        rows = a["slots"].long()
        have = torch.arange(before.shape[2], device=dev) < a["lengths"][rows][:, None]  # those that had a mass before
        gain = torch.where(have[:, None], (a["mass"] - before)[rows], 0.0)
        assert a["mass"].isfinite().all() and gain.min() >= 0
        assert (gain.amax((1, 2)) <= 2 * torch.tensor(lens, device=dev) + 1e-3).all()


@pytest.mark.parametrize("lens,had", [([1], [500]), ([1, 2], [3000, 40]), ([1] * 30, [17 * i for i in range(30)])])
@pytest.mark.parametrize("offset", [0.0, 900.0])
def test_masses_add_up(lens, had, offset):
    """Every token and query head hands out a weight of one, whatever its scores have in common (here up to 1e5)."""
    a = attention_inputs(lens, had, 4, 2, 128, BF, dev, tracked=True, behind=0.0)
    a["mass"].zero_()
    a["cos"] = a["sin"] = None
    for name, heads in (("q", 4), ("k", 2)):
        a[name].view(-1, heads, 128)[..., 0] = offset
    a["k_cache"][..., 0] = offset
    ops.cached_attention(**a)
    rows = a["slots"].long()
    have = torch.arange(a["mass"].shape[2], device=dev) < (a["lengths"][rows] + torch.tensor(lens, device=dev))[:, None]
    total = torch.where(have[:, None], a["mass"][rows].double(), 0.0).sum(-1)
    want = 2.0 * torch.tensor(lens, dtype=torch.float64, device=dev)[:, None]
    # sums of thousands of weights in 32 bits, and the denominators' reciprocal and the hardware's exp2 (2^-22 each)
    assert ((total / want - 1).abs() <= 1e-5).all(), float((total / want - 1).abs().max())


@pytest.mark.parametrize("D,H,Hk", [(96, 6, 2), (128, 3, 3), (128, 8, 1)])
@pytest.mark.parametrize("scale", [2.0, 30.0, 1e9])
def test_large_scales_of_other_heads(D, H, Hk, scale):
    """Scales on both sides of the one from which products are rounded first, with the other head dims and groups."""
    for lens, had, prefix in SHAPES:
        a = attention_inputs(lens, had, H, Hk, D, BF, dev, prefix=prefix)
        check_attention(ops.cached_attention, {**a, "cos": None, "sin": None, "sm_scale": scale}, HALF)
