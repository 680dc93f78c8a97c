"""The plain forms of the cache operators against definitions in 64 bits, and the refusals that need no GPU."""
import math

import pytest
import torch

from atomic_ai_hybrid_b200 import ops
from _cache import BF, F32, F64, attention_inputs, check_attention, copied, evict_truth, extreme_scores, gen, score_truth

CPU = torch.device("cpu")


@pytest.mark.parametrize("dtype", [F32, F64, BF])
@pytest.mark.parametrize("lens,had,heads,prefix", [
    ([1], [0], (2, 2, 8), None), ([3, 1, 5], [4, 0, 9], (4, 2, 8), None), ([1, 1, 1], [7, 2, 0], (6, 2, 16), ([5], [0, 0, 0])),
    ([2, 4, 0, 1, 3], [0, 3, 5, 1, 2], (3, 1, 8), ([6, 2], [0, 1, 1, -1, 0]))])
def test_plain_attention(dtype, lens, had, heads, prefix):
    a = attention_inputs(lens, had, *heads, dtype, CPU, prefix=prefix, tracked=True)
    check_attention(ops.cached_attention, a, torch.finfo(dtype).eps / 2 if dtype == BF else 0.0)


def test_plain_attention_forms():
    a = attention_inputs([2, 2, 2], [3, 0, 1], 2, 1, 8, F32, CPU)
    y, _ = check_attention(ops.cached_attention, a, 0.0)
    b = {**copied(a), "cu_seqlens": None, **{n: a[n].view(3, 2, -1) for n in ("q", "k", "v")}}
    y3, _ = check_attention(ops.cached_attention, b, 0.0)
    assert torch.equal(y.view(3, 2, -1), y3)
    with pytest.raises(ValueError, match="cu_seqlens"):
        ops.cached_attention(**{**b, "cu_seqlens": a["cu_seqlens"]})
    one = attention_inputs([1, 1], [3, 2], 2, 2, 8, F32, CPU)
    check_attention(ops.cached_attention, {**one, "cu_seqlens": None}, 0.0)
    check_attention(ops.cached_attention, {**one, "cos": None, "sin": None, "sm_scale": 0.3}, 0.0)
    check_attention(ops.cached_attention, {**one, "seen": one["lengths"] * 0 + 1}, 0.0)


def test_plain_attention_padding():
    """Sequences that cannot run give zeros and write nothing."""
    a = attention_inputs([2, 2, 2, 2], [3, 0, 1, 2], 2, 2, 8, F32, CPU, prefix=([4], [0, 0, 0, 0]), tracked=True)
    S = a["k_cache"].shape[0]
    for slot in (-1, S, 2 ** 31 - 1):
        b = copied(a)
        b["slots"][1] = slot
        y, _ = check_attention(ops.cached_attention, b, 0.0)
        assert (y[2:4] == 0).all() and (y[:2] != 0).any()
    for name, value in (("lengths", -1), ("lengths", a["k_cache"].shape[2] - 1), ("lengths", 2 ** 31 - 1), ("seen", -1),
                        ("seen", a["cos"].shape[0] - 1), ("seen", 2 ** 31 - 1)):
        b = copied(a)
        b["seen"] = b["lengths"] + 4
        b[name][b["slots"][2]] = value
        y, _ = check_attention(ops.cached_attention, b, 0.0)
        assert (y[4:6] == 0).all() and (y[6:] != 0).any()
    for value in (-1, S, a["k_cache"].shape[2] + 1):  # no prefix, or one whose length makes no sense
        b = copied(a)
        if value > S:
            b["lengths"][b["prefix"][0]] = value
        else:
            b["prefix"][:] = value
        check_attention(ops.cached_attention, b, 0.0)


@pytest.mark.parametrize("keep,recent,n", [(1, 0, 2), (4, 2, 9), (4, 4, 5), (6, 1, 6), (3, 0, 12)])
def test_plain_evict(keep, recent, n):
    g = gen(keep, CPU)
    S, Hk, M, D = 4, 3, 13, 4
    kc, vc = torch.randn(S, Hk, M, D, generator=g), torch.randn(S, Hk, M, D, generator=g)
    mass = torch.randint(0, 4, (S, Hk, M), generator=g).float()
    mass[0, 0, :3] = torch.tensor([math.nan, math.inf, -math.inf])
    held = torch.rand(S, Hk, M, generator=g).argsort(-1).to(torch.int32)
    lengths = torch.tensor([n, n, max(0, n - 2), M + 1], dtype=torch.int32)
    seen = torch.full((S,), M, dtype=torch.int32)
    for slots in (None, torch.tensor([2, 0, -1, S], dtype=torch.int32)):
        args = [t.clone() for t in (kc, vc, mass, held)]
        want = evict_truth(kc, vc, mass, held, lengths, seen, keep, recent, slots)
        assert ops.cache_evict(*args, lengths, seen, keep, recent=recent, slots=slots) is None
        for x, y in zip(args, want):
            assert torch.equal(x.nan_to_num(99.0), y.nan_to_num(99.0))


@pytest.mark.parametrize("keep,recent", [(0, 0), (3, 4), (3, -1)])
def test_evict_refuses(keep, recent):
    z = torch.zeros(1, 1, 4, 8)
    with pytest.raises(ValueError, match="cache_evict: keep"):
        ops.cache_evict(z, z.clone(), z[..., 0], z[..., 0].int(), torch.tensor([4], dtype=torch.int32),
                        torch.tensor([4], dtype=torch.int32), keep, recent=recent)


def _scores(R, V, dtype, seed=0):
    g = gen(seed, CPU)
    x = (torch.randn(R, V, generator=g) * 3).to(dtype)
    y = torch.randint(0, V, (R,), generator=g)
    return x, y


@pytest.mark.parametrize("temperature", [1.0, 0.5, 3.0])
def test_plain_logprobs_and_gradient(temperature):
    x, y = _scores(9, 17, F64)
    y[2], y[5] = -100, 17
    x[0, :5] = -math.inf
    x[1] = -math.inf
    x[3, 4] = math.nan
    x[4] = math.nan
    x[6, y[6]] = -math.inf
    x[7] = 0.25
    x.requires_grad_()
    out = ops.token_logprobs(x, y, top=6, temperature=temperature)
    want = score_truth(x.detach(), y, 6, temperature)
    for got, w in zip(out, want):
        assert (got == w).all() if not got.dtype.is_floating_point else torch.allclose(got, w, rtol=1e-12, atol=1e-12)
    assert out[0][1] == -math.inf and out[1][1] == 0 and (out[2][1] == -1).all() and out[0][2] == 0 and out[0][5] == 0
    assert out[2][7].tolist() == [0, 1, 2, 3, 4, 5]
    g, ge = torch.randn(9, dtype=F64, generator=gen(1, CPU)), torch.randn(9, dtype=F64, generator=gen(2, CPU))
    dx, = torch.autograd.grad(out[:2], [x], [g, ge])
    assert torch.allclose(dx, score_truth(x.detach(), y, 0, temperature, g, ge)[-1], rtol=1e-12, atol=1e-12)
    assert (dx[1] == 0).all() and (dx[4] == 0).all() and dx.isfinite().all()


def test_logprobs_gradient_by_differences():
    x, y = _scores(4, 7, F64, seed=3)
    y[1] = -100
    assert torch.autograd.gradcheck(lambda t: ops.token_logprobs(t, y, temperature=0.7), [x.requires_grad_()])


def test_logprobs_refuses():
    x, y = _scores(3, 5, F32)
    for match, args, kw in [("one int64 token", (x, y[:2]), {}), ("one int64 token", (x, y.int()), {}),
                            ("one int64 token", (x[0], y), {}), ("top", (x, y), dict(top=6)), ("top", (x, y), dict(top=-1)),
                            ("top", (torch.zeros(3, 100), y), dict(top=65)), ("temperature", (x, y), dict(temperature=0.0)),
                            ("temperature", (x, y), dict(temperature=math.inf)), ("temperature", (x, y), dict(temperature=math.nan))]:
        with pytest.raises(ValueError, match=match):
            ops.token_logprobs(*args, **kw)


def test_token_scores_of_a_model():
    """Log-probabilities and entropies of labels through a model, and their gradients against the log-softmax's."""
    from atomic_ai_hybrid_b200.config import get_preset
    from atomic_ai_hybrid_b200.models import HybridMoEModel
    from atomic_ai_hybrid_b200.training.loss import token_scores

    torch.manual_seed(0)
    cfg = get_preset("tiny", num_layers=2, vocab_size=300)
    model = HybridMoEModel(cfg, compute_dtype=F32)
    ids = torch.randint(0, 300, (2, 65), generator=gen(1, CPU))
    batch = {"input_ids": ids[:, :-1], "labels": ids[:, 1:].clone()}
    batch["labels"][0, :10] = -100

    def grads(f):
        model.zero_grad()
        lp, entropy = f()
        (lp.sum() * 0.1 + 0.01 * entropy.sum()).backward()
        return lp.detach(), entropy.detach(), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}

    def plain():
        h, _ = model(batch["input_ids"])
        logp = torch.log_softmax(h @ model.lm_weight().t(), -1)
        given = batch["labels"] >= 0
        lp = logp.gather(2, batch["labels"].clamp(min=0)[..., None])[..., 0] * given
        return lp, -(logp.exp() * logp).sum(-1)

    a, b = grads(lambda: token_scores(model, batch, chunk=50)), grads(plain)
    assert a[0].shape == batch["labels"].shape and (a[0][0, :10] == 0).all()
    for x, y in zip(a[:2], b[:2]):
        assert torch.allclose(x, y, rtol=1e-4, atol=1e-4)
    assert set(a[2]) == set(b[2])
    for n in a[2]:
        assert (a[2][n] - b[2][n]).norm() <= 1e-3 * b[2][n].norm() + 1e-6, n
    with torch.no_grad():
        assert torch.allclose(token_scores(model, batch)[0], a[0], atol=1e-5)


def test_launches_counted():
    from atomic_ai_hybrid_b200.utils.counters import LaunchCounter

    c = LaunchCounter()
    c.enable()
    q, cache = torch.zeros(4, 128), torch.zeros(4, 1, 8, 64)

    def count(L=1, cu=None, prefix=None, mass=None, rows=4):
        c.reset()
        c.add("cached_attention", (q[:rows], None, None, cache, cache, None, None, None, L, cu, None, prefix, None, mass, None, 1.0))
        return c.count

    some = torch.zeros(3, dtype=torch.int32)
    assert count() == 3 and count(L=4) == 3 and count(L=5) == 5 and count(cu=some) == 5 and count(prefix=some) == 4
    assert count(mass=some) == 4 and count(cu=some, mass=some) == 7 and count(prefix=some, mass=some) == 6
    assert count(rows=0) == 0 and count(cu=some[:1]) == 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_plain_logprobs_extremes(dtype):
    for x, y, T in extreme_scores(dtype, CPU):
        out, want = ops.token_logprobs(x, y, top=3, temperature=T), score_truth(x, y, 3, T)
        for i in (0, 1, 3):
            assert torch.allclose(out[i].double(), want[i].clamp(min=torch.finfo(F32).min), rtol=3e-5, atol=3e-5), (T, i)
        assert torch.equal(out[2], want[2])
    for T in (1e-38, 1e38, -1.0):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_logprobs(x, y, temperature=T)


def test_evict_slot_given_twice():
    g = gen(0, CPU)
    k, v = (torch.randn(3, 2, 40, 8, generator=g) for _ in range(2))
    mass, held = torch.rand(3, 2, 40, generator=g), torch.arange(40, dtype=torch.int32).expand(3, 2, 40).contiguous()
    n, seen = torch.full((3,), 40, dtype=torch.int32), torch.full((3,), 40, dtype=torch.int32)
    want = evict_truth(k, v, mass, held, n, seen, 12, 4, torch.tensor([2, 0]))
    ops.cache_evict(k, v, mass, held, n, seen, 12, recent=4, slots=torch.tensor([2, 0, 2, -1, 0], dtype=torch.int32))
    assert all(torch.equal(a, b) for a, b in zip((k, v, mass, held), want))


def test_token_scores_of_no_tokens():
    from atomic_ai_hybrid_b200.training.loss import token_scores

    class Nothing:
        def __call__(self, ids, return_hidden):
            return torch.zeros(*ids.shape, 8), []

        def lm_weight(self):
            return torch.zeros(30, 8)

    ids = torch.zeros(0, 5, dtype=torch.long)
    assert [tuple(t.shape) for t in token_scores(Nothing(), {"input_ids": ids, "labels": ids})] == [(0, 5), (0, 5)]
