"""sm_100a kernels of the cache operators (cached_attention, cache_evict, token_logprobs) against their definitions in 64
bits; ``_cache.py`` derives the bounds."""
import math

import pytest
import torch

from atomic_ai_hybrid_b200 import ops
from _cache import BF, F32, attention_inputs, attention_truth, check_attention, copied, evict_truth, extreme_scores, gen, offsets, score_truth

pytestmark = pytest.mark.gpu
dev = "cuda"
HALF = 2.0 ** -8  # half a step of bf16


# ------------------------------------------------------------------ cached_attention
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("lens,had", [([1], [0]), ([1], [1000]), ([1, 1, 1], [15, 16, 17]), ([2, 1, 0, 7], [31, 0, 5, 300]),
                                      ([16, 17, 33], [0, 1, 127]), ([200, 1, 130], [0, 700, 64]), ([1] * 40, list(range(0, 800, 20)))])
def test_attention_sizes(D, lens, had):
    for H, Hk in ((1, 1), (6, 3), (8, 1)):
        check_attention(ops.cached_attention, attention_inputs(lens, had, H, Hk, D, BF, dev, tracked=True), HALF)


@pytest.mark.parametrize("lens,had,prefix", [
    ([1] * 5, [0, 3, 90, 1, 20], ([700], [0] * 5)),
    ([1] * 9, [5] * 9, ([33, 257], [0, 0, 1, 1, 1, -1, 0, 0, 1])),        # runs, a conversation without, the first prefix again
    ([3, 0, 5, 1], [0, 0, 2, 9], ([64], [0, 0, 0, 0])),
    ([150, 40, 1, 300], [0, 10, 0, 0], ([500], [0, 0, 0, -1])),
    ([1] * 200, [i % 7 for i in range(200)], ([130], [0] * 200)),
    ([1] * 3, [4, 4, 4], ([0], [0, 0, 0]))])                              # an empty prefix
@pytest.mark.parametrize("H,Hk,D", [(4, 4, 128), (6, 2, 64), (16, 1, 96)])
def test_attention_prefix(lens, had, prefix, H, Hk, D):
    a = attention_inputs(lens, had, H, Hk, D, BF, dev, prefix=prefix, tracked=len(lens) < 20)
    check_attention(ops.cached_attention, a, HALF)
    if all(n == 1 for n in lens):
        check_attention(ops.cached_attention, {**a, "cu_seqlens": None}, HALF)


def test_attention_long_rows():
    check_attention(ops.cached_attention, attention_inputs([1, 5], [40000, 9], 2, 2, 128, BF, dev, tracked=True), HALF)
    check_attention(ops.cached_attention, attention_inputs([1500], [700], 2, 1, 128, BF, dev, tracked=True), HALF)
    check_attention(ops.cached_attention, attention_inputs([1000, 3], [0, 1], 3, 3, 64, BF, dev, prefix=([2000], [0, 0])), HALF)


def test_attention_forms():
    """Batches of rows, rows of one token, no tables, a scale, positions of one's own."""
    a = attention_inputs([3, 3, 3, 3], [0, 4, 100, 33], 4, 2, 128, BF, dev, tracked=True)
    y, _ = check_attention(ops.cached_attention, a, HALF)
    b = {**copied(a), "cu_seqlens": None, **{n: a[n].view(4, 3, -1) for n in ("q", "k", "v")}}
    y3, _ = check_attention(ops.cached_attention, b, HALF)
    assert torch.equal(y.view(4, 3, -1), y3)
    check_attention(ops.cached_attention, {**a, "cos": None, "sin": None, "sm_scale": 0.02}, HALF)
    check_attention(ops.cached_attention, {**a, "seen": a["lengths"] * 0 + 7}, HALF)
    check_attention(ops.cached_attention, {**a, "slots": None, "lengths": a["lengths"].clamp(max=5)}, HALF)
    check_attention(ops.cached_attention, {**a, "sm_scale": 0.0}, HALF)  # equal weights
    check_attention(ops.cached_attention, {**a, "sm_scale": -0.1}, HALF)
    none = ops.cached_attention(**{**copied(a), **{n: a[n][:0] for n in ("q", "k", "v")}, "cu_seqlens": offsets([0] * 4, dev)})
    assert none.shape == (0, 4 * 128)


def test_attention_strides():
    """Column slices of a projection, at 16-byte boundaries and off them, rows that overlap nothing."""
    a = attention_inputs([1, 40, 3], [60, 2, 17], 4, 2, 64, BF, dev)
    want, _ = check_attention(ops.cached_attention, a, HALF)
    T = a["q"].shape[0]
    for off in (0, 8, 1, 3):
        wide = torch.full((T, 4 * 64 + 2 * 2 * 64 + 11), math.nan, device=dev, dtype=BF)
        at, views = off, {}
        for n in ("q", "k", "v"):
            w = a[n].shape[1]
            wide[:, at:at + w] = a[n]
            views[n] = wide[:, at:at + w]
            at += w
        assert torch.equal(ops.cached_attention(**{**copied(a), **views}), want)


def test_attention_rows_of_no_sequence():
    """Rows before the first and behind the last sequence come out as zeros, offsets out of range are cut."""
    a = attention_inputs([4, 2], [5, 30], 2, 2, 64, BF, dev)
    for n in ("q", "k", "v"):
        a[n] = torch.cat([a[n][:3] * math.nan, a[n], a[n][:2] * math.nan])
    a["cu_seqlens"] = a["cu_seqlens"] + 3
    y, _ = check_attention(ops.cached_attention, a, HALF)
    assert (y[:3] == 0).all() and (y[9:] == 0).all()
    b = copied(a)
    b["cu_seqlens"] = torch.tensor([-5, 7, 100], dtype=torch.int32, device=dev)
    b["lengths"].clamp_(max=2)
    for n in ("q", "k", "v"):
        b[n] = b[n].nan_to_num(0.5)
    c = {**copied(b), "cu_seqlens": torch.tensor([0, 7, 11], dtype=torch.int32, device=dev)}
    assert torch.equal(ops.cached_attention(**b), ops.cached_attention(**c))
    assert (ops.cached_attention(**{**copied(a), "cu_seqlens": offsets([], dev), "slots": a["slots"][:0]}) == 0).all()


def test_attention_padding():
    a = attention_inputs([2, 2, 20, 2], [3, 0, 1, 2], 2, 2, 64, BF, dev, prefix=([40], [0, 0, 0, 0]), tracked=True)
    S, M = a["k_cache"].shape[0], a["k_cache"].shape[2]
    for slot in (-1, S, 2 ** 31 - 1, -2 ** 31):
        for i in (0, 1, 2, 3):
            b = copied(a)
            b["slots"][i] = slot
            y, _ = check_attention(ops.cached_attention, b, HALF)
            first = int(a["cu_seqlens"][i])
            assert (y[first:int(a["cu_seqlens"][i + 1])] == 0).all()
    for name, value in (("lengths", -1), ("lengths", M - 1), ("lengths", 2 ** 31 - 1), ("seen", -1), ("seen", a["cos"].shape[0] - 1),
                        ("seen", 2 ** 31 - 1)):
        b = copied(a)
        b["seen"] = b["lengths"] + 40
        b[name][b["slots"][1]] = value
        y, _ = check_attention(ops.cached_attention, b, HALF)
        assert (y[2:4] == 0).all() and (y[4:] != 0).any()
    for value in (-1, S, 2 ** 31 - 1):
        b = copied(a)
        b["prefix"][1:3] = value
        check_attention(ops.cached_attention, b, HALF)
    for rows in (-3, M + 1):
        b = copied(a)
        b["lengths"][b["prefix"][0]] = rows
        check_attention(ops.cached_attention, b, HALF)
    b = copied(a)
    b["slots"][:] = -1
    y, _ = check_attention(ops.cached_attention, b, HALF)
    assert (y == 0).all()


@pytest.mark.parametrize("behind", [math.nan, math.inf, -math.inf, torch.finfo(BF).min])
@pytest.mark.parametrize("lens,had", [([1, 3], [9, 200]), ([140, 1], [3, 5])])
def test_attention_behind_the_rows(behind, lens, had):
    """What the cache holds behind its rows reaches nothing."""
    a = attention_inputs(lens, had, 2, 2, 128, BF, dev, behind=behind, prefix=([37], [0, 0]), tracked=True)
    y, _ = check_attention(ops.cached_attention, a, HALF)
    assert y.isfinite().all()


def test_attention_clips_and_extremes():
    """Infinite and NaN inputs are clipped like the layers', large scores leave one weight, equal ones the mean."""
    a = attention_inputs([5, 130], [20, 7], 2, 2, 64, BF, dev)
    for n in ("q", "k", "v"):
        a[n][1, :5] = torch.tensor([math.nan, math.inf, -math.inf, 5e3, -1e30], device=dev)
        a[n][90, 3] = math.nan
    b = {**copied(a), "cos": None, "sin": None, "sm_scale": 2.0 ** -20}
    y, c = check_attention(ops.cached_attention, b, HALF)
    assert y.isfinite().all() and c["k_cache"][a["slots"][0].long(), 0, 21, :5].tolist() == [0, 1000, -1000, 1000, -1000]
    for scale in (30.0, -30.0):  # scores of thousands: bf16 queries and keys, so the products are exact in what the check reads
        b = {**attention_inputs([5, 130], [200, 7], 2, 2, 64, BF, dev), "cos": None, "sin": None, "sm_scale": scale}
        y, _ = check_attention(ops.cached_attention, b, HALF)
    rising = attention_inputs([1, 200], [3000, 0], 1, 1, 64, BF, dev, std=0.0)
    rising["q"][:, 0] = 1.0
    rising["cos"] = rising["sin"] = None
    rising["k_cache"][rising["slots"][0].long(), 0, :3000, 0] = torch.linspace(-900, 900, 3000, device=dev).to(BF)
    check_attention(ops.cached_attention, rising, HALF)
    check_attention(ops.cached_attention, {**rising, "sm_scale": -1.0}, HALF)


def test_attention_offsets_past_32_bits():
    """A cache of more than 2^32 bytes and 2^31 values: slots at its end."""
    S, Hk, M, D = 5, 16, 262150, 128
    assert S * Hk * M * D > 2 ** 31
    small = attention_inputs([1, 3], [70, 0], 16, 16, D, BF, dev, extra=0, behind=0.0)
    kc = torch.zeros(S, Hk, M, D, device=dev, dtype=BF)
    vc = torch.zeros(S, Hk, M, D, device=dev, dtype=BF)
    rows = small["k_cache"].shape[2]
    for i, s in enumerate((4, 3)):
        kc[s, :, :rows] = small["k_cache"][small["slots"][i].long()]
        vc[s, :, :rows] = small["v_cache"][small["slots"][i].long()]
    lengths = torch.tensor([0, 0, 0, 0, 70], dtype=torch.int32, device=dev)
    big = {**copied(small), "k_cache": kc, "v_cache": vc, "lengths": lengths, "slots": torch.tensor([4, 3], dtype=torch.int32, device=dev)}
    want = copied(small)
    y, z = ops.cached_attention(**want), ops.cached_attention(**big)
    assert torch.equal(y, z)
    assert torch.equal(kc[4, :, 70], want["k_cache"][small["slots"][0].long(), :, 70])
    # rows at the end of a long slot
    lengths[4] = M - 8
    big["seen"] = lengths.clamp(max=20)
    small["lengths"].zero_()
    y, z = ops.cached_attention(**copied(small)), ops.cached_attention(**big)  # a slot of zeros before the new rows
    assert z.isfinite().all() and (kc[4, :, M - 8] != 0).any() and (kc[4, :, M - 7:] == 0).all()


def _step(a, H, Hk, D, seed):
    g = gen(seed, dev)
    B = a["slots"].numel()
    return {n: torch.randn(B, h * D, generator=g, device=dev).to(BF) for n, h in (("q", H), ("k", Hk), ("v", Hk))}


def test_attention_captured_and_on_other_streams():
    """Captured steps replayed with new inputs and lengths, two graphs in turn, eager calls between them, another stream."""
    H, Hk, D = 4, 2, 128
    make = lambda s: attention_inputs([1] * 6, [3, 100, 40, 0, 7, 513], H, Hk, D, BF, dev, prefix=([90], [0] * 6), tracked=True, seed=s)  # noqa: E731
    graphs = []
    for seed in (0, 1):
        a = {**make(seed), "cu_seqlens": None}
        eager = copied(a)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.cached_attention(**copied(a))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.cached_attention(**a)
            a["lengths"].index_add_(0, a["slots"].long(), torch.ones_like(a["slots"]))
        graphs.append((graph, a, out, eager))
    for turn in range(3):
        for i, (graph, a, out, eager) in enumerate(graphs):
            new = _step(a, H, Hk, D, 10 * turn + i)
            for n, t in new.items():
                a[n].copy_(t)
                eager[n] = t
            graph.replay()
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                want = ops.cached_attention(**eager)
                eager["lengths"].index_add_(0, eager["slots"].long(), torch.ones_like(eager["slots"]))
            torch.cuda.current_stream().wait_stream(s)
            assert torch.equal(out, want)
            for n in ("mass", "held", "lengths"):
                assert torch.equal(a[n], eager[n])
            for n in ("k_cache", "v_cache"):
                assert torch.equal(a[n].nan_to_num(5.0), eager[n].nan_to_num(5.0))


def test_attention_repeats_exactly():
    """The same call gives the same bits, however its work is cut."""
    for lens, had, pre in (([1] * 30, [50 * i for i in range(30)], None), ([700, 3], [5, 900], ([400], [0, 0]))):
        a = attention_inputs(lens, had, 8, 4, 128, BF, dev, prefix=pre, tracked=True)
        b, c = copied(a), copied(a)
        assert torch.equal(ops.cached_attention(**b), ops.cached_attention(**c))
        assert torch.equal(b["mass"], c["mass"])


def test_attention_types_without_kernels():
    for D, dtype in ((32, BF), (64, F32), (256, F32)):
        check_attention(ops.cached_attention, attention_inputs([3, 1], [4, 9], 2, 1, D, dtype, dev, prefix=([5], [0, 0]), tracked=True),
                        HALF if dtype == BF else 0.0)


def test_attention_refusals():
    a = attention_inputs([2, 1], [3, 4], 4, 2, 64, BF, dev, prefix=([5], [0, 0]), tracked=True)

    def refused(match, **kw):
        with pytest.raises((RuntimeError, ValueError), match=match):
            ops.cached_attention(**{**copied(a), **kw})

    refused("q and the caches must be bf16", q=a["q"].float())
    refused("k must", k=a["k"][:, :64])
    refused("v must", v=a["v"].float())
    refused("do not make heads", q=a["q"][:, :192])
    refused("k_cache and v_cache", v_cache=a["v_cache"][:, :1])
    refused("k_cache and v_cache", k_cache=a["k_cache"].transpose(1, 2))
    refused("different tensors", v_cache=(same := a["k_cache"].clone()), k_cache=same)
    refused("k_cache and v_cache", v_cache=a["v_cache"].cpu())
    refused("lengths", lengths=a["lengths"].long())
    refused("lengths", lengths=a["lengths"][:2])
    refused("come together", sin=None)
    refused("cos must", cos=a["cos"][:, :32])
    refused("sin must", sin=a["sin"][:3])
    refused("cos must", cos=a["cos"].to(BF))
    refused("mass and held come together", held=None)
    refused("mass", mass=a["mass"][:1])
    refused("held", held=a["held"].long())
    refused("prefix", prefix=a["prefix"][:1])
    refused("seen", seen=a["lengths"][:1])
    refused("slots", slots=a["slots"].long())
    refused("sm_scale", sm_scale=math.nan)
    refused("16-byte", k_cache=torch.zeros(a["k_cache"].numel() + 1, device=dev, dtype=BF)[1:].view(a["k_cache"].shape))
    refused("need a state slot", slots=None, cu_seqlens=offsets([0] * 50, dev), prefix=None)


# ------------------------------------------------------------------ cache_evict
def _evict_inputs(S, Hk, M, D, dtype=BF, seed=0, levels=None):
    g = gen(seed, dev)
    caches = [torch.randn(S, Hk, M, D, generator=g, device=dev).to(dtype) for _ in range(2)]
    mass = torch.rand(S, Hk, M, generator=g, device=dev).exp() if levels is None else \
        torch.randint(0, levels, (S, Hk, M), generator=g, device=dev).float() - 1
    held = torch.rand(S, Hk, M, generator=g, device=dev).argsort(-1).to(torch.int32)
    return caches + [mass, held]


def _check_evict(args, lengths, seen, keep, recent, slots=None):
    want = evict_truth(*args, lengths, seen, keep, recent, slots)
    got = [t.clone() for t in args]
    ops.cache_evict(*got, lengths, seen, keep, recent=recent, slots=slots)
    for name, x, y in zip(("k", "v", "mass", "held"), got, want):
        assert torch.equal(x.nan_to_num(77.0), y.nan_to_num(77.0)), name
    return got


@pytest.mark.parametrize("M,n,keep,recent", [(9, 9, 8, 0), (9, 8, 1, 1), (700, 600, 300, 40), (700, 513, 512, 512), (1030, 1025, 20, 3),
                                             (3000, 2999, 2500, 0), (3000, 2048, 64, 64)])
@pytest.mark.parametrize("levels", [None, 4, 1])
def test_evict_sizes(M, n, keep, recent, levels):
    S = 5
    lengths = torch.tensor([n, max(0, n - 1), keep, 0, M + 1], dtype=torch.int32, device=dev)
    seen = torch.full((S,), M, dtype=torch.int32, device=dev)
    for D, dtype in ((64, BF), (96, BF), (128, BF), (4, F32)):
        args = _evict_inputs(S, 3, M, D, dtype, levels=levels)
        _check_evict(args, lengths, seen, keep, recent)
    order = torch.tensor([1, -1, 0, S, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    _check_evict(args, lengths, seen, keep, recent, order)


def test_evict_special_masses():
    S, M, keep = 2, 300, 100
    args = _evict_inputs(S, 2, M, 64)
    m = args[2]
    m[0, 0] = math.nan
    m[0, 1] = math.inf
    m[1, 0, ::2], m[1, 0, 1::2] = 0.0, -0.0
    m[1, 1, ::3], m[1, 1, 1::3], m[1, 1, 2::3] = -math.inf, math.nan, -1e38
    lengths, seen = torch.full((S,), M, dtype=torch.int32, device=dev), torch.full((S,), M, dtype=torch.int32, device=dev)
    for recent in (0, 30):
        _check_evict(args, lengths, seen, keep, recent)
    seen[:] = -2 ** 31  # every row is new: the lowest stay
    got = _check_evict(args, lengths, seen, keep, 30)
    assert torch.equal(got[3][..., :keep], args[3][..., :keep])


def test_evict_rows_past_shared_memory():
    M, n = 60000, 59990
    args = _evict_inputs(1, 2, M, 64, levels=50)
    lengths, seen = torch.tensor([n], dtype=torch.int32, device=dev), torch.tensor([M], dtype=torch.int32, device=dev)
    for keep, recent in ((30000, 500), (59989, 0), (16, 16)):
        _check_evict(args, lengths, seen, keep, recent)


def test_evict_captured_and_nothing_to_do():
    args = _evict_inputs(3, 2, 200, 64)
    lengths, seen = torch.full((3,), 200, dtype=torch.int32, device=dev), torch.full((3,), 200, dtype=torch.int32, device=dev)
    want = [t.clone() for t in args]
    ops.cache_evict(*want, lengths, seen, 50, recent=10)
    live = [t.clone() for t in args]
    ops.cache_evict(*[t.clone() for t in args], lengths, seen, 50, recent=10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_evict(*live, lengths, seen, 50, recent=10)
    for _ in range(2):
        for t, s in zip(live, args):
            t.copy_(s)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(live, want))
    for keep, slots in ((200, None), (500, None), (50, torch.zeros(0, dtype=torch.int32, device=dev))):
        same = [t.clone() for t in args]
        ops.cache_evict(*same, lengths, seen, keep, slots=slots)
        assert all(torch.equal(x, y) for x, y in zip(same, args))


def test_evict_refusals():
    k, v, m, h = _evict_inputs(2, 2, 20, 64)
    n = torch.full((2,), 20, dtype=torch.int32, device=dev)
    for match, args, kw in [("keep", (k, v, m, h, n, n, 0), {}), ("keep", (k, v, m, h, n, n, 5), dict(recent=6)),
                            ("mass", (k, v, m[:1], h, n, n, 5), {}), ("mass", (k, v, m.double(), h, n, n, 5), {}),
                            ("held", (k, v, m, h.long(), n, n, 5), {}), ("lengths", (k, v, m, h, n[:1], n, 5), {}),
                            ("seen", (k, v, m, h, n, n.long(), 5), {}), ("k_cache and v_cache", (k, v[:, :1], m, h, n, n, 5), {}),
                            ("different tensors", (k, k, m, h, n, n, 5), {}),
                            ("slots", (k, v, m, h, n, n, 5), dict(slots=torch.zeros(2, dtype=torch.int64, device=dev)))]:
        with pytest.raises((RuntimeError, ValueError), match=match):
            ops.cache_evict(*args, **kw)


def test_tokens_tracked_and_thinned_out():
    """A conversation's steps with a budget: rows gather attention, the cache is cut, later tokens answer from what is left."""
    H, Hk, D, budget, slack = 4, 2, 64, 40, 8
    a = attention_inputs([30, 55], [0, 0], H, Hk, D, BF, dev, tracked=True, extra=1)
    M = a["k_cache"].shape[2]
    a["cos"], a["sin"] = (torch.cat([t, t, t]) for t in (a["cos"], a["sin"]))
    a["seen"] = a["lengths"].clone()
    _, a = check_attention(ops.cached_attention, a, HALF)
    rows = a["slots"].long()
    a["lengths"][rows] += torch.tensor([30, 55], dtype=torch.int32, device=dev)
    a["seen"][rows] += torch.tensor([30, 55], dtype=torch.int32, device=dev)
    a["cu_seqlens"] = None
    for t in range(25):
        if int(a["lengths"].max()) >= min(M, budget + slack):
            state = [a[n] for n in ("k_cache", "v_cache", "mass", "held")]
            for n, x in zip(("k_cache", "v_cache", "mass", "held"), _check_evict(state, a["lengths"], a["seen"], budget, slack, a["slots"])):
                a[n] = x
            a["lengths"].clamp_(max=budget)
            for i in range(2):  # the newest tokens are all there
                s, seen = int(rows[i]), int(a["seen"][rows[i]])
                have = a["held"][s, :, :int(a["lengths"][s])]
                assert all(set(range(seen - slack, seen)) <= set(have[h].tolist()) for h in range(Hk))
        a.update(_step(a, H, Hk, D, 100 + t))
        _, a = check_attention(ops.cached_attention, a, HALF)
        a["lengths"][rows] += 1
        a["seen"][rows] += 1


# ------------------------------------------------------------------ token_logprobs
def _scores(R, V, dtype, seed=0, std=3.0):
    g = gen(seed, dev)
    x = (torch.randn(R, V, generator=g, device=dev) * std).to(dtype)
    return x, torch.randint(0, V, (R,), generator=g, device=dev)


def _check_scores(x, y, top=0, temperature=1.0, grad=True):
    """fp32 sums of at most 10^5 values over 512 threads (200 additions each, 2^-24 a step, 1.2e-5 relative), hardware exp2
    and log2 (2^-21): 3e-5 on a sum of weights, and so on a log-probability; entropies and gradients carry it once more
    with their size.  A bf16 gradient is rounded by 2^-8."""
    want = score_truth(x.detach(), y, top, temperature)
    leaf = x.detach().requires_grad_(grad)
    out = ops.token_logprobs(leaf, y, top=top, temperature=temperature)
    assert len(out) == (4 if top else 2)
    for i in (0, 1) + ((3,) if top else ()):
        assert out[i].dtype == F32
        fin = want[i].isfinite()
        assert torch.equal(out[i].isfinite(), fin)
        assert (out[i] == want[i].float())[~fin].all()
        err = (out[i].double() - want[i]).abs()[fin]
        # log p = (x - max) / T - log sum: each of the two rounded
        assert (err <= 3e-5 * (1 + want[i].abs()[fin])).all(), (i, float(err.max()))
    if top:
        assert out[2].dtype == torch.int64 and torch.equal(out[2], want[2])
    if grad:
        g, ge = torch.randn(len(y), generator=gen(5, dev), device=dev), torch.randn(len(y), generator=gen(6, dev), device=dev)
        dx, = torch.autograd.grad(out[:2], [leaf], [g, ge])
        w = score_truth(x.detach(), y, 0, temperature, g, ge)[-1]
        x64 = x.detach().double()
        size = (g.abs() + ge.abs() * (1 + want[1].float())).double()[:, None] / temperature
        tol = (2.0 ** -8 if x.dtype == BF else 0) * w.abs() + 1e-4 * size * (w.abs() / size).clamp(max=1.0) + 1e-7 * size
        assert dx.dtype == x.dtype and dx.shape == x.shape
        assert ((dx.double() - w).abs() <= tol).all(), float(((dx.double() - w).abs() - tol).max())
        del x64
    return out


@pytest.mark.parametrize("R,V", [(1, 1), (2, 2), (3, 31), (5, 300), (4, 4096), (1, 50304), (3, 50305), (2, 151936), (160, 1000), (300, 513)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_sizes(R, V, dtype):
    x, y = _scores(R, V, dtype, seed=R + V)
    for top, T in ((0, 1.0), (min(V, 5), 1.0), (min(V, 64), 0.7), (1, 4.0)):
        _check_scores(x, y, top, T)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("top", [1, 7, 64])
def test_logprobs_orders(dtype, top):
    """Logits in rising and falling order, all equal, a few large ones side by side, only a few with a probability."""
    V = 60000
    up = torch.linspace(-30, 30, V, device=dev)
    rows = [up, up.flip(0), torch.zeros(V, device=dev), torch.full((V,), -2.5, device=dev)]
    block = torch.zeros(V, device=dev)
    block[30000:30000 + 2000] = torch.linspace(5, 25, 2000, device=dev)
    stripe = torch.full((V,), -math.inf, device=dev)   # what every thread of one eighth of a warp reads
    stripe[(torch.arange(V, device=dev) // 64) % 64 == 3] = 1.0
    few = torch.full((V,), -math.inf, device=dev)
    few[[5, 59999, 777]] = torch.tensor([1.0, 1.0, 2.0], device=dev)
    x = torch.stack(rows + [block, stripe, few]).to(dtype)
    y = torch.tensor([V - 1, 0, 17, 5, 31999, 192, 777], device=dev)
    out = _check_scores(x, y, top)
    assert out[2][6].tolist() == ([777, 5, 59999] + [-1] * 61)[:top]
    assert out[2][2].tolist() == list(range(top))


def test_logprobs_special_values():
    low = torch.finfo(BF).min
    x, y = _scores(12, 3001, BF, seed=3)
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 777] = -5.0
    x[3] = low
    x[4, ::2] = math.nan
    x[5, y[5]] = -math.inf
    x[6, y[6]] = math.nan
    x[7, :1500] = -math.inf
    x[8] *= 1000
    y[9], y[10], y[11] = -100, 3001, 2 ** 40
    for T in (1.0, 0.3):
        out = _check_scores(x, y, 4, T)
        assert (out[0][:2] == -math.inf).all() and (out[1][:3] == 0).all() and (out[2][:2] == -1).all()
        assert out[2][2].tolist() == [777, -1, -1, -1] and (out[0][5:7] == -math.inf).all() and (out[0][9:] == 0).all()
        assert out[2][3].tolist() == [0, 1, 2, 3]
    z, t = _scores(2, 500, F32)
    z[0, [7, 90]] = math.inf   # the largest finite number: the two of them share the mass
    z[1, 3] = 1e30
    lp, H, index, best = ops.token_logprobs(z, torch.tensor([7, 3], device=dev), top=2)
    assert index[0].tolist() == [7, 90] and abs(float(lp[0]) + math.log(2)) < 1e-6 and abs(float(H[0]) - math.log(2)) < 1e-6
    assert float(lp[1]) == 0 and float(H[1]) == 0
    for V in (100, 5000):  # near a large common value nothing is lost
        z = torch.randn(3, V, generator=gen(1, dev), device=dev) + 9000
        _check_scores(z, torch.zeros(3, dtype=torch.long, device=dev), 3)


def test_logprobs_strides():
    """Row strides and starts off 16 bytes, gradients of expanded weights."""
    for dtype in (BF, F32):
        for off, V in ((0, 1000), (1, 1001), (3, 777), (8, 2048)):
            wide = torch.full((6, V + 13), math.nan, device=dev, dtype=dtype)
            x, y = _scores(6, V, dtype, seed=V)
            wide[:, off:off + V] = x
            view = wide[:, off:off + V]
            a, b = ops.token_logprobs(x, y, top=3), ops.token_logprobs(view, y, top=3)
            assert torch.equal(a[2], b[2])
            _check_scores(view, y, 3)
            leaf = wide.clone().requires_grad_()
            lp, H = ops.token_logprobs(leaf[:, off:off + V], y)
            (lp.sum() + 0.1 * H.mean()).backward()
            ones = torch.ones(6, device=dev)
            w = score_truth(x, y, 0, 1.0, ones, ones * 0.1 / 6)[-1]
            assert ((leaf.grad[:, off:off + V].double() - w).abs() <= (2.0 ** -8 if dtype == BF else 1e-4) * w.abs() + 1e-6).all()


def test_logprobs_captured():
    """Forward and backward in a graph, replayed with new logits."""
    x, y = _scores(40, 3000, F32)
    x.requires_grad_()
    g = torch.randn(40, device=dev)

    def both():
        lp, H, index, best = ops.token_logprobs(x, y, top=3)
        return lp, H, index, best, torch.autograd.grad([lp, H], [x], [g, 0.1 * g])[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in (4, 5):
        with torch.no_grad():
            x.copy_(_scores(40, 3000, F32, seed=seed)[0])
        graph.replay()
        for a, b in zip(out, both()):
            assert torch.equal(a, b)


def test_logprobs_one_output_alone():
    x, y = _scores(5, 400, F32)
    x.requires_grad_()
    one = torch.ones(5, device=dev)
    for i in (0, 1):
        dx, = torch.autograd.grad(ops.token_logprobs(x, y)[i].sum(), [x])
        w = score_truth(x.detach(), y, 0, 1.0, one * (i == 0), one * (i == 1))[-1]
        assert ((dx.double() - w).abs() <= 1e-4 * w.abs() + 1e-6).all()
    out = ops.token_logprobs(x, y, top=2)
    assert not out[2].requires_grad and not out[3].requires_grad
    assert not ops.token_logprobs(x.detach(), y)[0].requires_grad
    empty = ops.token_logprobs(torch.zeros(0, 9, device=dev), torch.zeros(0, dtype=torch.long, device=dev), top=2)
    assert [tuple(t.shape) for t in empty] == [(0,), (0,), (0, 2), (0, 2)]


def test_logprobs_refusals():
    x, y = _scores(4, 50, BF)
    for match, args, kw in [("one int64 token", (x, y[:3]), {}), ("one int64 token", (x, y.int()), {}), ("top", (x, y), dict(top=51)),
                            ("top", (x.repeat(1, 3), y), dict(top=65)), ("temperature", (x, y), dict(temperature=-1.0)),
                            ("temperature", (x, y), dict(temperature=1e-60)), ("expected bf16 or fp32", (x.half(), y), {}),
                            ("tokens", (x, y.cpu()), {}), ("unit channel stride", (x.repeat(1, 2)[:, ::2], y), {})]:
        with pytest.raises((RuntimeError, ValueError), match=match):
            ops.token_logprobs(*args, **kw)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_extremes(dtype):
    """Temperatures so small that a masked place's exponent would be infinite, and logits so large."""
    for x, y, T in extreme_scores(dtype, dev):
        _check_scores(x, y, 3, T, grad=False)
        out = ops.token_logprobs(x.requires_grad_(), y, temperature=T)
        dx, = torch.autograd.grad(out[0].sum() + out[1].sum(), [x])
        assert dx.isfinite().all()


@pytest.mark.parametrize("M", [300, 60000])
def test_evict_slot_given_twice(M):
    args = _evict_inputs(3, 2, M, 64, levels=40)
    n, seen = torch.full((3,), M, dtype=torch.int32, device=dev), torch.full((3,), M, dtype=torch.int32, device=dev)
    want = evict_truth(*args, n, seen, 100, 20, torch.tensor([2, 0]))
    ops.cache_evict(*args, n, seen, 100, recent=20, slots=torch.tensor([2, 0, 2, 2, -1, 0], dtype=torch.int32, device=dev))
    assert all(torch.equal(a, b) for a, b in zip(args, want))


@pytest.mark.parametrize("D", [64, 96, 128])
def test_attention_tables_between_boundaries(D):
    """Rotation tables that start between 16-byte boundaries, for few and for many rows."""
    a = attention_inputs([1, 40], [30, 20], 4, 2, D, BF, dev)
    for name in ("cos", "sin"):
        odd = torch.zeros(a[name].numel() + 1, device=dev)[1:].view(a[name].shape)
        a[name] = odd.copy_(a[name])
    check_attention(ops.cached_attention, a, HALF)


def test_attention_refuses_too_many_heads():
    a = attention_inputs([1], [3], 4, 2, 64, BF, dev)
    a["q"] = torch.zeros(1, 2 * 129 * 64, device=dev, dtype=BF)
    with pytest.raises((RuntimeError, ValueError), match="128 query heads"):
        ops.cached_attention(**a)
    a["q"] = torch.zeros(1, 256, device=dev, dtype=BF)
    with pytest.raises((RuntimeError, ValueError), match="sm_scale"):
        ops.cached_attention(**a, sm_scale=1e300)


def test_attention_128_heads_share_one():
    """The most query heads of one key head: single tokens, a prompt, a prefix."""
    for lens, kept, kw in [([1, 1], [50, 7], {}), ([9], [100], {}), ([1, 3], [5, 6], dict(prefix=([70], [0, 0])))]:
        check_attention(ops.cached_attention, attention_inputs(lens, kept, 128, 1, 64, BF, dev, **kw), HALF)


@pytest.mark.parametrize("lens,kept,kw", [([900], [300], {}), ([300, 40, 1], [0, 10, 700], dict(prefix=([1500], [0, 0, 0]))),
                                          ([1, 7], [1000, 1200], {})])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_loses_no_more_than_two_roundings(lens, kept, kw, D):
    """Values in no common direction: the weights' rounding and the output's, each at most 2^-8 / sqrt(3) of the output on
    average, add up to sqrt(2 / 3) 2^-8; queries, scores and sums keep 32 bits."""
    a = attention_inputs(lens, kept, 8, 4, D, BF, dev, **kw)
    o = attention_truth(**copied(a))[0]
    y = ops.cached_attention(**copied(a)).double().reshape(o.shape)
    assert (y - o).norm() <= (2 / 3) ** 0.5 * 2.0 ** -8 * o.norm(), float((y - o).norm() / o.norm())


@pytest.mark.parametrize("H,Hk", [(99, 3), (14, 2), (6, 2), (40, 8)])
def test_attention_repeats_where_heads_do_not_fill_a_tile(H, Hk):
    """Rows of a tile that belong to no query hold what was there before: the same call, with other ones between, gives the same bits."""
    a = attention_inputs([15, 1, 0, 6, 22, 200], [0, 0, 229, 408, 0, 31], H, Hk, 96, BF, dev, prefix=([119, 340], [-1, 1, 1, 0, -1, 1]), std=4.0)
    b = attention_inputs([700], [100], 16, 4, 128, BF, dev, std=30.0, seed=1)
    first, _ = check_attention(ops.cached_attention, a, HALF)
    for _ in range(10):
        ops.cached_attention(**copied(b))
        assert torch.equal(ops.cached_attention(**copied(a)), first)
