"""sm_100a kernels of the stateful serving operators (selective_scan, gdn2_recurrent, sample) against
their definitions in 64 bits.

Bounds, from the arithmetic: a state takes at most about 4 roundings of 2^-24 per token on top of the
decay's (one unit in the last place), and forgets with 1 - e^{-0.01}; 6 * 2^-24 / 0.00995 = 3.6e-5 of
the largest state value bounds what adds up.  The hardware's exp, log and divide enter the inputs with
about 2^-21.  A bf16 result adds its rounding, 2^-8 of the value at most."""
import math

import pytest
import torch

from atomic_ai_hybrid_b200 import ops
from atomic_ai_hybrid_b200.ops import reference as R

pytestmark = pytest.mark.gpu
dev = "cuda"
BF, F32 = torch.bfloat16, torch.float32
REL = 4e-5


def _gen(seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(dev, torch.int32)


def _d(v):
    if isinstance(v, (list, tuple)):
        return [_d(t) for t in v]
    return v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v


# ------------------------------------------------------------------ selective_scan
def _scan_inputs(lens, C, P, N, dtype, seed=0, pool=None, wdtype=F32, bias=True):
    g = _gen(seed)
    T, pool = sum(lens), pool or len(lens) + 2
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    xz = r(T, 2 * C).to(dtype)
    return dict(x=xz[:, C:], dt=(r(T, C) - 2.5).to(dtype), A=-torch.rand(C // P, generator=g, device=dev) * 15 - 1,
                Bm=r(T, N).to(dtype), Cm=r(T, N).to(dtype), conv_w=(r(C, 4) * 0.5).to(wdtype),
                conv_b=r(C) * 0.1 if bias else None, conv_state=r(pool, 3, C).to(dtype), state=r(pool, C // P, P, N),
                slots=torch.randperm(pool, generator=g, device=dev)[:len(lens)].to(torch.int32))


def _check_scan(a, cu, call=None):
    """Runs the kernel and the 64-bit form on copies of the states and compares everything."""
    ref = {k: _d(v) for k, v in a.items()}
    ref["conv_state"], ref["state"] = ref["conv_state"].clone(), ref["state"].clone()
    y64 = R.selective_scan(**ref, cu_seqlens=cu)
    y = (call or (lambda: ops.selective_scan(**a, cu_seqlens=cu)))()
    C = a["x"].shape[-1]
    top = ref["state"].abs().max().clamp(min=1.0)
    assert torch.equal(a["conv_state"].double(), ref["conv_state"])
    assert ((a["state"].double() - ref["state"]).abs() <= REL * top).all()
    assert y.dtype == a["x"].dtype and y.shape == a["x"].shape
    tol = REL * top * ref["Cm"].abs().sum(-1, keepdim=True)
    if y.dtype == BF:
        tol = tol + 2.0 ** -8 * y64.abs()
    assert ((y.double() - y64).abs() <= tol).all(), ((y.double() - y64).abs() - tol).max()
    return y, C


@pytest.mark.parametrize("C,P,N", [(2048, 64, 128), (1536, 192, 128), (256, 64, 64), (128, 64, 32), (40, 8, 64), (24, 24, 128), (7, 7, 32)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_tokens(C, P, N, dtype):
    a = _scan_inputs([1] * 5, C, P, N, dtype, seed=C + N)
    _check_scan(a, None)


@pytest.mark.parametrize("lens", [[1], [2], [3], [15], [16], [17], [33], [0, 5, 0, 1, 70], [129, 64, 1, 255], [300], [1100, 3, 513], [1, 2, 3, 0, 15, 16, 17, 31, 32, 33, 200]])
@pytest.mark.parametrize("C,P,N,dtype", [(256, 64, 128, BF), (192, 192, 64, BF), (72, 8, 32, BF), (21, 7, 128, BF), (64, 64, 128, F32)])
def test_scan_prompts(lens, C, P, N, dtype):
    a = _scan_inputs(lens, C, P, N, dtype, seed=sum(lens) + C)
    _check_scan(a, _cu(lens))


def test_scan_long_prompt():
    """Many segments: the state is handed from one to the next."""
    lens = [5000, 1, 2500]
    _check_scan(_scan_inputs(lens, 512, 64, 128, BF, seed=3), _cu(lens))


@pytest.mark.parametrize("N", [32, 64, 128])
def test_scan_strong_decays(N):
    """Steps and rates from no decay to the -20 clamp at every token, side by side."""
    lens = [45, 700, 64]
    a = _scan_inputs(lens, 256, 8, N, BF, seed=12)
    a["A"] = -torch.logspace(-3, 2, 32, device=dev)[torch.randperm(32, generator=_gen(1), device=dev)].contiguous()
    a["dt"] = (torch.randn(sum(lens), 256, generator=_gen(2), device=dev) * 4).to(BF)
    # A = -1e-3 forgets with 1 - e^{-1e-5}: no room for REL there, but 700 tokens take 700 * 6 * 2^-24 at most
    ref = {k: _d(v) for k, v in a.items()}
    ref["conv_state"], ref["state"] = ref["conv_state"].clone(), ref["state"].clone()
    y64 = R.selective_scan(**ref, cu_seqlens=_cu(lens))
    y = ops.selective_scan(**a, cu_seqlens=_cu(lens))
    top = ref["state"].abs().max()
    rel = 700 * 6 * 2.0 ** -24
    assert ((a["state"].double() - ref["state"]).abs() <= rel * top).all()
    assert ((y.double() - y64).abs() <= 2.0 ** -8 * y64.abs() + rel * top * ref["Cm"].abs().sum(-1, keepdim=True)).all()


def test_scan_padded_and_strided_inputs():
    """(B, L, C) tokens, inputs that are columns of wider rows, bf16 taps, no bias."""
    B, L, C, N = 3, 37, 128, 64
    a = _scan_inputs([L] * B, C, 64, N, BF, seed=9, wdtype=BF, bias=False)
    wide = torch.randn(B * L, 3 * N + 5, device=dev, generator=_gen(1)).to(BF)
    a["Bm"], a["Cm"] = wide[:, 3:3 + N], wide[:, N + 7:2 * N + 7]
    shaped = {k: v.unflatten(0, (B, L)) if k in ("x", "dt", "Bm", "Cm") else v for k, v in a.items()}
    _check_scan(a, _cu([L] * B), call=lambda: ops.selective_scan(**shaped).flatten(0, 1))


def test_scan_in_parts_equals_whole():
    """A prompt given in pieces, the last of single tokens, ends where the whole prompt does."""
    L, C, N = 150, 256, 128
    a = _scan_inputs([L], C, 64, N, BF, seed=11)
    b = {k: v.clone() if k in ("conv_state", "state") else v for k, v in a.items()}
    whole = ops.selective_scan(**a, cu_seqlens=_cu([L]))
    parts, at = [], 0
    for n in (100, 2, 45, 1, 1, 1):
        piece = {k: v[at:at + n] if k in ("x", "dt", "Bm", "Cm") else v for k, v in b.items()}
        parts.append(ops.selective_scan(**piece, cu_seqlens=_cu([n])))
        at += n
    assert torch.equal(a["conv_state"], b["conv_state"])
    top = a["state"].abs().max().clamp(min=1.0)
    assert ((a["state"] - b["state"]).abs() <= 2 * REL * top).all()
    tol = 2.0 ** -7 * whole.double().abs() + 2 * REL * top * a["Cm"].double().abs().sum(-1, keepdim=True)
    assert ((torch.cat(parts).double() - whole.double()).abs() <= tol).all()


@pytest.mark.parametrize("lens", [[1, 1, 1], [40, 3, 200]])
def test_scan_padding_slots(lens):
    """A slot outside the state gives zeros and leaves every state alone."""
    a = _scan_inputs(lens, 128, 64, 64, BF, seed=2)
    for bad in (-1, a["state"].shape[0], 1 << 30):
        b = {k: v.clone() if isinstance(v, torch.Tensor) and k in ("conv_state", "state", "slots") else v for k, v in a.items()}
        b["slots"][1] = bad
        keep = b["state"].clone(), b["conv_state"].clone()
        y = ops.selective_scan(**b, cu_seqlens=_cu(lens))
        assert (y[lens[0]:lens[0] + lens[1]] == 0).all()
        untouched = torch.ones(keep[0].shape[0], dtype=torch.bool, device=dev)
        untouched[b["slots"][[0, 2]].long()] = False
        assert torch.equal(b["state"][untouched], keep[0][untouched])
        assert torch.equal(b["conv_state"][untouched], keep[1][untouched])
        assert not torch.equal(b["state"][~untouched], keep[0][~untouched])


@pytest.mark.parametrize("L", [1, 3, 100])
def test_scan_extreme_values(L):
    """Infinities, NaN and huge values are clipped as the layer clips them; steps at both clamps."""
    a = _scan_inputs([L], 64, 64, 64, BF, seed=5)
    x, dt = a["x"].clone(), a["dt"].clone()
    x[0, 0], x[0, 1], x[-1, 2] = 1e30, -1e30, 3e4
    dt[0, 3], dt[0, 4], dt[-1, 5], dt[0, 6] = math.nan, math.inf, -math.inf, 60.0
    a["x"], a["dt"] = x, dt
    a["Bm"][0, 0], a["Bm"][0, 1], a["Cm"][0, 2], a["Cm"][-1, 3] = math.nan, math.inf, -math.inf, math.nan
    a["A"][:] = -50.0  # dt A far below the -20 clamp
    ref = {k: _d(v) for k, v in a.items()}
    ref["conv_state"], ref["state"] = ref["conv_state"].clone(), ref["state"].clone()
    y64 = R.selective_scan(**ref, cu_seqlens=_cu([L]))
    y = ops.selective_scan(**a, cu_seqlens=_cu([L]))
    assert torch.isfinite(y).all() and torch.isfinite(a["state"]).all()
    # channels differ by 1e6 in size here: each is held to its own largest input (u <= 1e3, B <= 1e3)
    assert ((a["state"].double() - ref["state"]).abs() <= REL * 1e6).all()
    assert ((y.double() - y64).abs() <= 2.0 ** -8 * y64.abs() + REL * 1e6 * 1e3 * 64).all()
    small = torch.arange(64, device=dev) >= 8  # ordinary channels with the clipped B: u <= 10
    assert ((a["state"].double() - ref["state"]).abs()[a["slots"].long()][0, 0, small] <= REL * 1e4).all()


@pytest.mark.parametrize("A", [-0.05, -3.0, -5.0])
def test_scan_largest_values(A):
    """Every input at its clip, decays on both sides of the change from blocks to single tokens (A dt = 3.3 a token):
    nothing overflows, and errors stay in proportion to the sums of absolute values."""
    L = 90
    a = _scan_inputs([L], 64, 64, 128, BF, seed=6)
    sign = lambda t, s: torch.where(torch.rand(t.shape, generator=_gen(s), device=dev) < 0.5, -1.0, 1.0).to(BF)  # noqa: E731
    a["x"], a["dt"] = sign(a["x"], 1) * 1e30, torch.full_like(a["dt"], 60.0)
    a["Bm"], a["Cm"], a["A"][:] = sign(a["Bm"], 2) * 1e4, sign(a["Cm"], 3) * 1e4, A
    ref = {k: _d(v) for k, v in a.items()}
    ref["conv_state"], ref["state"] = ref["conv_state"].clone(), ref["state"].clone()
    y64 = R.selective_scan(**ref, cu_seqlens=_cu([L]))
    y = ops.selective_scan(**a, cu_seqlens=_cu([L]))
    most = 1e6 / -math.expm1(A)  # of a state
    assert torch.isfinite(y).all()
    assert ((a["state"].double() - ref["state"]).abs() <= REL * most).all()
    assert ((y.double() - y64).abs() <= 2.0 ** -8 * y64.abs() + REL * most * 128e3).all()


@pytest.mark.parametrize("N", [32, 64, 128])
@pytest.mark.parametrize("form,dtype", [("one each", BF), ("one each", F32), ("offsets", BF), ("offsets", F32), ("block", BF)])
def test_scan_growth(N, form, dtype):
    """Rates above zero grow the state up to infinity, in every form alike (the layer's are below zero)."""
    rates = torch.tensor([1.0, 20.0, 60.0, 87.9, 88.3, 88.6, 95.0, 300.0], device=dev)
    a = _scan_inputs([1] * 3, 64, 8, N, dtype, seed=8)
    a["A"], a["dt"] = rates, torch.full_like(a["dt"], 60.0)  # a step of 1
    cu = None if form == "one each" else _cu([1] * 3)
    if form == "block":  # each token first of 16 whose steps are the smallest, 1e-9 of its growth
        lead = {n: a[n][:, None].repeat(1, 16, 1).flatten(0, 1) for n in ("x", "dt", "Bm", "Cm")}
        lead["dt"].unflatten(0, (3, 16))[:, 1:] = -100.0
        a.update(lead)
        cu = _cu([16] * 3)
    lo = dict(dt_min=1e-9) if form == "block" else {}
    ref = {k: _d(v) for k, v in a.items()}
    ref["conv_state"], ref["state"] = ref["conv_state"].clone(), ref["state"].clone()
    R.selective_scan(**ref, cu_seqlens=cu, **lo)
    ops.selective_scan(**a, cu_seqlens=cu, **lo)
    # the last two factors are beyond the floats' end themselves, whatever they multiply
    want, got = ref["state"].float(), a["state"]
    mine = a["slots"].long()
    want[mine, 6:] = want[mine, 6:].sign() * math.inf
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got.sign(), want.sign())
    finite = torch.isfinite(want)
    assert ((got - want).abs()[finite] <= REL * want.abs()[finite].clamp(min=10.0)).all()


def test_scan_bad_offsets_stay_in_bounds():
    """Offsets outside the rows or in the wrong order never reach outside the buffers."""
    lens = [20, 30]
    a = _scan_inputs(lens, 128, 64, 64, BF, seed=7)
    canary = a["state"].clone()
    for cu in ([-5, 20, 9000], [40, 10, 50], [0, 1 << 30, 3]):
        ops.selective_scan(**a, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    other = torch.ones(canary.shape[0], dtype=torch.bool, device=dev)
    other[a["slots"].long()] = False
    assert torch.equal(a["state"][other], canary[other])


def _poisoned(shape, dtype):
    """Leaves NaN in the memory that the next output of this shape takes; returns its address."""
    t = torch.full(shape, math.nan, device=dev, dtype=dtype)
    return t.data_ptr()


# offsets of 60 rows that leave rows uncovered at either end, in falling order, out of range, or have no sequence
OPEN = [[0, 20, 50], [7, 20, 60], [3, 3, 40], [60, 60, 60], [0, 0, 0], [9], [40, 10, 50], [0, 50, 20], [50, 30, 10], [-5, 20, 9000]]


@pytest.mark.parametrize("cu", OPEN)
@pytest.mark.parametrize("form", ["blocks", "blocks of any width", "tokens"])
def test_scan_rows_of_no_sequence_are_zero(cu, form):
    T, C = 60, 21 if form == "blocks of any width" else 80
    a = _scan_inputs([T // 2] * 2, C, C, 64, F32 if form == "tokens" else BF, seed=4)
    a["slots"] = a["slots"][:len(cu) - 1].contiguous()
    cu_dev = torch.tensor(cu, dtype=torch.int32, device=dev)
    ref = {k: _d(v) for k, v in a.items()}
    ref["conv_state"], ref["state"] = ref["conv_state"].clone(), ref["state"].clone()
    want = R.selective_scan(**ref, cu_seqlens=cu_dev)
    at = _poisoned(a["x"].shape, a["x"].dtype)
    y = ops.selective_scan(**a, cu_seqlens=cu_dev)
    assert y.data_ptr() == at and torch.isfinite(y).all()
    if all(s <= e for s, e in zip(cu, cu[1:])):  # falling offsets promise finite values only
        assert (y[(want == 0).all(1)] == 0).all()
        assert (y.double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()


def test_scan_open_rows_beside_many_sequences():
    """More rows than blocks that clear them, more sequences than a warp looks at together, cut and whole."""
    for lens, T in (([1] * 70, 900), ([40, 0, 3] * 25, 9000), ([3000, 500], 12000)):
        a = _scan_inputs([T], 64, 64, 32, BF, seed=5, pool=len(lens) + 2)
        a["slots"] = torch.randperm(len(lens) + 2, generator=_gen(1), device=dev)[:len(lens)].to(torch.int32)
        head = 33
        cu = (_cu(lens) + head).contiguous()
        used = {k: v[head:head + sum(lens)] if k in ("x", "dt", "Bm", "Cm") else v.clone() if "state" in k else v
                for k, v in a.items()}
        want = ops.selective_scan(**used, cu_seqlens=_cu(lens))
        at = _poisoned(a["x"].shape, BF)
        y = ops.selective_scan(**a, cu_seqlens=cu)
        assert y.data_ptr() == at
        assert (y[:head] == 0).all() and (y[head + sum(lens):] == 0).all()
        # cut elsewhere, the same sums in another order
        assert (y[head:head + sum(lens)].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()


def test_scan_on_another_stream_and_empty():
    a = _scan_inputs([64, 2], 256, 64, 128, BF, seed=8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _check_scan(a, _cu([64, 2]))
    torch.cuda.current_stream().wait_stream(s)
    e = _scan_inputs([0], 128, 64, 64, BF)
    assert ops.selective_scan(**e, cu_seqlens=_cu([0])).shape == (0, 128)
    rows = {k: v.unflatten(0, (2, 0)) if k in ("x", "dt", "Bm", "Cm") else v for k, v in _scan_inputs([0, 0], 128, 64, 64, BF).items()}
    assert ops.selective_scan(**rows).shape == (2, 0, 128)


def test_calls_repeat_themselves():
    """The same call on the same states gives the same bits, cut into segments or not."""
    for lens in ([1] * 5, [3, 9, 1], [700, 17, 1, 333], [4000]):
        first = None
        for _ in range(3):
            a, b = _scan_inputs(lens, 256, 64, 128, BF, seed=2), _gdn_inputs([min(l, 40) for l in lens], 2, 128, BF, seed=2)
            now = (ops.selective_scan(**a, cu_seqlens=_cu(lens)), a["state"], a["conv_state"],
                   ops.gdn2_recurrent(**b, cu_seqlens=_cu([min(l, 40) for l in lens])), b["state"], b["conv_state"])
            first = first or now
            assert all(torch.equal(s, t) for s, t in zip(first, now))


@pytest.mark.parametrize("lens,dtype,kernels", [([1] * 3, BF, 1), ([5, 3], BF, 1), ([40, 40], BF, 2), ([3000], BF, 4), ([64], F32, 1)])
def test_scan_launches_are_counted(lens, dtype, kernels):
    """The launch counter's figure is the number of kernels in the call's CUDA graph."""
    from cuda.bindings import runtime
    from atomic_ai_hybrid_b200.utils.counters import launch_counter

    a, cu = _scan_inputs(lens, 256, 64, 128, dtype, seed=1), _cu(lens)
    ops.selective_scan(**a, cu_seqlens=cu)
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before, was = launch_counter.count, launch_counter.on
    launch_counter.enable()
    with torch.cuda.graph(graph):
        ops.selective_scan(**a, cu_seqlens=cu)
    counted = launch_counter.count - before
    if not was:
        launch_counter.disable()
    launch_counter.count = before
    handle = graph.raw_cuda_graph()
    _, _, n = runtime.cudaGraphGetNodes(handle)
    _, nodes, _ = runtime.cudaGraphGetNodes(handle, n)
    kinds = [runtime.cudaGraphNodeGetType(node)[1] for node in nodes]
    assert kinds.count(runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel) == kernels
    assert counted == kernels


def test_scan_refusals():
    a = _scan_inputs([4], 128, 64, 64, BF)
    cu = _cu([4])

    def refused(match, **kw):
        with pytest.raises((RuntimeError, ValueError), match=match):
            ops.selective_scan(**{**a, "cu_seqlens": cu, **kw})

    refused("dt must", dt=a["dt"].float())
    refused("dt must", dt=a["dt"][:, :64])
    refused("B must", Bm=a["Bm"][:2])
    refused("state must", state=a["state"].to(BF))
    refused("do not make", state=a["state"][:, :, :32].contiguous())
    refused("conv_state", conv_state=a["conv_state"].float())
    refused("conv_w", conv_w=a["conv_w"][:64].contiguous())
    refused("A must", A=a["A"].double())
    refused("cu_seqlens", cu_seqlens=cu.long())
    refused("slots", slots=a["slots"].long())
    refused("slots", slots=torch.zeros(3, dtype=torch.int32, device=dev))
    refused("slot each", cu_seqlens=None, slots=None, state=a["state"][:1], conv_state=a["conv_state"][:1])
    refused("cu_seqlens packs", x=a["x"][None])


# ------------------------------------------------------------------ gdn2_recurrent
def _gdn_inputs(lens, H, D, dtype, seed=0, wdtype=BF, bias=True):
    g = _gen(seed)
    T, d, pool = sum(lens), H * D, len(lens) + 2
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    wide = r(T, 6 * d + 8).to(dtype)
    cols = {n: wide[:, i * d:(i + 1) * d] for i, n in enumerate("qkvbwf")}
    return dict(**cols, conv_w=[(r(d, 4) * 0.5).to(wdtype) for _ in range(3)],
                conv_b=[r(d) * 0.1 if bias else None for _ in range(3)], decay_a=r(H) * 0.5 - 1.0,
                conv_state=r(pool, 3, 3, d).to(dtype), state=r(pool, H, D, D) * 0.1,
                slots=torch.randperm(pool, generator=g, device=dev)[:len(lens)].to(torch.int32))


def _check_gdn(a, cu):
    ref = {k: _d(v) for k, v in a.items()}
    ref["conv_state"], ref["state"] = ref["conv_state"].clone(), ref["state"].clone()
    o64 = R.gdn2_recurrent(**ref, cu_seqlens=cu)
    o = ops.gdn2_recurrent(**a, cu_seqlens=cu)
    D = a["state"].shape[-1]
    top = ref["state"].abs().max().clamp(min=1.0)
    assert torch.equal(a["conv_state"].double(), ref["conv_state"])
    # k and q have norm 1 and the gates stay below 1, so h enters n and o with a factor of at most sqrt(D)
    assert ((a["state"].double() - ref["state"]).abs() <= REL * top).all()
    tol = REL * top * math.sqrt(D)
    if o.dtype == BF:
        tol = tol + 2.0 ** -8 * o64.abs()
    assert o.dtype == a["q"].dtype and o.shape == a["q"].shape
    assert ((o.double() - o64).abs() <= tol).all()


@pytest.mark.parametrize("H,D", [(16, 128), (6, 128), (3, 96), (1, 64), (5, 64)])
@pytest.mark.parametrize("dtype,wdtype", [(BF, BF), (BF, F32), (F32, F32)])
def test_gdn_tokens(H, D, dtype, wdtype):
    _check_gdn(_gdn_inputs([1] * 4, H, D, dtype, seed=H * D, wdtype=wdtype), None)


@pytest.mark.parametrize("lens", [[1], [2], [3], [4], [0, 5, 1, 0, 9], [40, 2]])
@pytest.mark.parametrize("H,D", [(2, 128), (2, 96), (3, 64)])
def test_gdn_few_tokens(lens, H, D):
    _check_gdn(_gdn_inputs(lens, H, D, BF, seed=sum(lens), bias=D != 96), _cu(lens))


def test_gdn_large_batch():
    _check_gdn(_gdn_inputs([1] * 200, 4, 128, BF, seed=1), None)


def test_gdn_padding_slots_and_streams():
    a = _gdn_inputs([1, 3, 2], 2, 128, BF, seed=4)
    a["slots"][1] = -1
    before = a["state"].clone(), a["conv_state"].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o = ops.gdn2_recurrent(**a, cu_seqlens=_cu([1, 3, 2]))
    torch.cuda.current_stream().wait_stream(s)
    assert (o[1:4] == 0).all() and (o[0] != 0).any()
    idle = torch.ones(before[0].shape[0], dtype=torch.bool, device=dev)
    idle[a["slots"][[0, 2]].long()] = False
    assert torch.equal(a["state"][idle], before[0][idle]) and torch.equal(a["conv_state"][idle], before[1][idle])


@pytest.mark.parametrize("cu", OPEN)
def test_gdn_rows_of_no_sequence_are_zero(cu):
    a = _gdn_inputs([30, 30], 2, 64, BF, seed=4)
    a["slots"] = a["slots"][:len(cu) - 1].contiguous()
    cu_dev = torch.tensor(cu, dtype=torch.int32, device=dev)
    ref = {k: _d(v) for k, v in a.items()}
    ref["conv_state"], ref["state"] = ref["conv_state"].clone(), ref["state"].clone()
    want = R.gdn2_recurrent(**ref, cu_seqlens=cu_dev)
    at = _poisoned(a["q"].shape, BF)
    o = ops.gdn2_recurrent(**a, cu_seqlens=cu_dev)
    assert o.data_ptr() == at and torch.isfinite(o).all()
    if all(s <= e for s, e in zip(cu, cu[1:])):
        assert (o[(want == 0).all(1)] == 0).all()
        assert (o.double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()


def test_gdn_matches_chunked_scan():
    """The state after a prompt through the chunked training kernel continues in the token form."""
    B, L, H, D = 2, 128, 2, 128
    g = _gen(6)
    q, k, v, w, b = (torch.randn(B, L, H, D, generator=g, device=dev) for _ in range(5))
    q, k = R.safe_l2norm(q, 1e-12), R.safe_l2norm(k, 1e-12)
    f = torch.randn(B, L, H, D, generator=g, device=dev)
    decay = torch.full((H,), -1.0, device=dev)
    gl = -torch.exp(decay)[:, None] * torch.nn.functional.softplus(f)
    o, hf = ops.gdn2(q, k, v, torch.sigmoid(w), torch.sigmoid(b), gl, return_final=True)
    serial, h64 = R.gdn2_token_serial(q, k, v, gl, torch.sigmoid(b), torch.sigmoid(w))
    # the chunked kernel's operands are bf16 (2^-9 each); the token form starts from its state
    assert (hf - h64).norm() <= 2e-2 * h64.norm()


@pytest.mark.parametrize("lens", [[800], [70, 769, 1]])
def test_gdn_prompt_forms_hand_over(lens):
    """The two forms that a prompt can take in serving, the chunked scan of training and the token form, from the same
    projections and state; then single tokens on the state of either.  Against 64 bits: the token form keeps its own
    bound.  The chunked kernel multiplies bf16 operands (2^-9 each, a few in a row: 2e-2 of the state, as above); with
    unit keys and gates below 1 no later token makes an error of the state larger."""
    from atomic_ai_hybrid_b200 import get_preset
    from atomic_ai_hybrid_b200.models.mixers import GatedDeltaNet2
    from atomic_ai_hybrid_b200.serving.state import DecodeState, serving

    torch.manual_seed(0)
    cfg = get_preset("hybrid_1b", d_model=256, n_heads=2)
    with torch.device(dev):
        mod = GatedDeltaNet2(cfg)
        mod.compute_dtype = BF
    B, d, T, after = len(lens), 256, sum(lens), 6
    g = _gen(3)
    rows = [torch.randn(1, T + after * B, d, generator=g, device=dev).to(BF) for _ in range(6)]
    start = torch.randn(B, 3, 3, d, generator=g, device=dev).to(BF), torch.randn(B, 2, 128, 128, generator=g, device=dev) * 0.1
    par = dict(conv_w=[getattr(mod, f"{n}_conv_w").detach() for n in "qkv"],
               conv_b=[getattr(mod, f"{n}_conv_b").detach() for n in "qkv"], decay_a=mod.decay_a.detach())
    prompt, cu = [t[:, :T] for t in rows], _cu(lens)
    c64 = dict(conv=start[0].double(), state=start[1].double())
    o64 = R.gdn2_recurrent(*(t[0].double() for t in prompt), **_d(par), conv_state=c64["conv"], state=c64["state"], cu_seqlens=cu)

    def states(form):
        st = DecodeState(mod, B)
        c = st.layers[mod]
        c["conv"].copy_(start[0])
        c["state"].copy_(start[1])
        if form == "chunked":
            with torch.no_grad(), serving(st, list(range(B)), lens) as call:
                return c, call._gdn2_chunked(mod, c, prompt)
        return c, ops.gdn2_recurrent(*(t[0] for t in prompt), **par, conv_state=c["conv"], state=c["state"], cu_seqlens=cu)

    size = c64["state"].norm()
    for form, tol in (("tokens", REL), ("chunked", 2e-2)):
        c, o = states(form)
        s64 = {n: t.clone() for n, t in c64.items()}
        own = dict(conv=c["conv"].double(), state=c["state"].double())
        assert torch.equal(own["conv"], s64["conv"])
        print(f"[gdn prompt] {lens} {form}: state {(own['state'] - s64['state']).norm() / size:.1e}, outputs {(o - o64).norm() / o64.norm():.1e}")
        assert (own["state"] - s64["state"]).norm() <= tol * size
        assert (o - o64).norm() <= (tol + 2.0 ** -8) * o64.norm()
        for k in range(after):
            now = [t[0, T + k * B:T + (k + 1) * B] for t in rows]
            y = ops.gdn2_recurrent(*now, **par, conv_state=c["conv"], state=c["state"])
            truth = R.gdn2_recurrent(*_d(now), **_d(par), conv_state=s64["conv"], state=s64["state"])
            cont = R.gdn2_recurrent(*_d(now), **_d(par), conv_state=own["conv"], state=own["state"])
            assert ((y - cont).abs() <= 2.0 ** -8 * cont.abs() + REL * math.sqrt(128)).all()
            assert (y - truth).norm() <= 2.0 ** -8 * truth.norm() + tol * size
        assert torch.equal(c["conv"].double(), s64["conv"])
        assert ((c["state"] - own["state"]).abs() <= REL * own["state"].abs().max().clamp(min=1.0)).all()
        assert (c["state"] - s64["state"]).norm() <= tol * size


def test_gdn_refusals():
    a = _gdn_inputs([2], 2, 64, BF)
    cu = _cu([2])

    def refused(match, **kw):
        with pytest.raises((RuntimeError, ValueError), match=match):
            ops.gdn2_recurrent(**{**a, "cu_seqlens": cu, **kw})

    refused("k must", k=a["k"].float())
    refused("f must", f=a["f"][:, :64])
    refused("state must", state=a["state"].double())
    refused("do not make", state=a["state"][:, :1].contiguous())
    refused("conv_state", conv_state=a["conv_state"][:, :2].contiguous())
    refused("decay_a", decay_a=a["decay_a"][:1])
    refused("conv_w", conv_w=[a["conv_w"][0], a["conv_w"][1], a["conv_w"][2].float()])
    refused("slots", slots=a["slots"].long())


# ------------------------------------------------------------------ sample
def _check_sample(logits, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Every token must be kept with the thresholds eased by 2e-5, and win the race among the tokens kept
    with them tightened by 2e-5, by a score within 1e-4 (fp32 scores of size up to 100 carry 1e-5)."""
    tokens, logprobs = ops.sample(logits, noise, temperature, top_k, top_p, min_p)
    B, V = logits.shape
    l = logits.double()
    l = torch.where(torch.isnan(l), -math.inf, l).clamp(max=torch.finfo(F32).max)
    col = lambda v, d: (v if isinstance(v, torch.Tensor) else torch.full((B,), v)).to(dev, d)[:, None]  # noqa: E731
    T, k, tp, mp = col(temperature, torch.float64), col(top_k, torch.long), col(top_p, torch.float64), col(min_p, torch.float64)
    greedy = ~(T > 0)
    k = torch.where(greedy, 1, torch.where(k <= 0, V, k))
    T = torch.where(greedy, 1.0, T)
    ranked, index = torch.sort(l, dim=1, descending=True, stable=True)
    nd = (ranked - ranked[:, :1]) / T
    mass = nd.exp()
    before = mass.cumsum(1) - mass
    rank = torch.arange(V, device=dev)[None]
    Z = mass.sum(1, keepdim=True)
    score = nd - noise.double().gather(1, index).log()

    def kept(ease):
        return ((rank < k) & ((rank == 0) | (before < (tp + ease) * Z)) & ((rank == 0) | (mass >= mp - ease))
                & (ranked > -math.inf))

    got = (index == tokens[:, None])
    assert tokens.dtype == torch.int64 and logprobs.dtype == F32
    assert (got.sum(1) == 1).all()
    assert (got & kept(2e-5)).any(1).all()
    mine = torch.where(got, score, 0.0).nan_to_num(0.0, -1e9, -1e9).sum(1)
    best = torch.where(kept(-2e-5), score, -math.inf).max(1).values
    assert (torch.isposinf(best) | (mine >= best - 1e-4)).all()
    logp = torch.where(got, nd, 0.0).sum(1) - Z[:, 0].log()
    assert ((logprobs.double() - logp).abs() <= 1e-5 * (1 + logp.abs())).all()
    return tokens


def _logits(B, V, dtype, seed, std=3.0):
    g = _gen(seed)
    return (torch.randn(B, V, generator=g, device=dev) * std).to(dtype), torch.empty(B, V, device=dev).exponential_(generator=g)


@pytest.mark.parametrize("B,V", [(1, 1), (2, 2), (3, 31), (5, 300), (4, 4096), (1, 50304), (3, 50305), (2, 151936), (160, 1000), (300, 513)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_sample_sizes(B, V, dtype):
    logits, noise = _logits(B, V, dtype, seed=B + V)
    _check_sample(logits, noise)
    _check_sample(logits, noise, temperature=0.8, top_k=50, top_p=0.9, min_p=0.02)


@pytest.mark.parametrize("kw", [dict(top_k=1), dict(top_k=2), dict(top_k=7, temperature=2.0), dict(top_p=0.0), dict(top_p=0.3),
                                dict(top_p=0.999), dict(min_p=0.3), dict(min_p=1.0), dict(temperature=0.0), dict(temperature=-1.0),
                                dict(temperature=0.05), dict(temperature=100.0, top_k=3), dict(top_k=10 ** 9),
                                dict(temperature=5.0, top_p=0.5, min_p=0.2, top_k=100)])
@pytest.mark.parametrize("std", [0.01, 4.0])
def test_sample_rules(kw, std):
    logits, noise = _logits(6, 5000, BF, seed=17, std=std)
    _check_sample(logits, noise, **kw)


def test_sample_ties():
    """Equal logits rank by index, equal scores go to the lowest index."""
    B, V = 4, 3000
    logits = torch.zeros(B, V, device=dev, dtype=BF)
    noise = torch.ones(B, V, device=dev)
    for kw in (dict(), dict(top_k=10), dict(top_p=0.5), dict(temperature=0.0)):
        assert (ops.sample(logits, noise, **kw)[0] == 0).all()
    noise[:, 9], noise[:, 20] = 0.5, 0.25
    assert (ops.sample(logits, noise, top_k=10)[0] == 9).all()
    assert (ops.sample(logits, noise, top_k=20)[0] == 9).all()
    assert (ops.sample(logits, noise, top_k=21)[0] == 20).all()
    assert (ops.sample(logits, noise)[0] == 20).all()


@pytest.mark.parametrize("kw", [dict(min_p=1.5), dict(min_p=math.nan), dict(top_p=0.0), dict(top_p=-1.0), dict(top_p=math.nan),
                                dict(top_p=math.nan, top_k=5), dict(min_p=2.0, top_p=0.5, top_k=7)])
@pytest.mark.parametrize("B,V", [(3, 3000), (1, 70000)])
def test_sample_rules_that_only_the_first_passes(kw, B, V):
    """Settings that no mass can meet keep the first token alone, not those as likely as it, and not all."""
    logits = torch.zeros(B, V, device=dev)
    logits[:, 7:40] = 3.0
    noise = torch.ones(B, V, device=dev)
    noise[:, 20] = 1e-9  # as likely as the first, and the winner of any race
    tokens, logprobs = ops.sample(logits, noise, temperature=0.9, **kw)
    want, wantp = R.sample(logits, noise, temperature=0.9, **kw)
    assert (tokens == 7).all() and torch.equal(tokens, want)
    assert ((logprobs - wantp).abs() <= 1e-5 * (1 + wantp.abs())).all()


def test_sample_masked_rows():
    low = torch.finfo(BF).min
    B, V = 7, 2000
    logits, noise = _logits(B, V, BF, seed=23)
    logits[0] = -math.inf                      # nothing left
    logits[1] = math.nan                       # nothing left
    logits[2] = -math.inf
    logits[2, 777] = -5.0                      # one left
    logits[3] = low                            # the lowest value everywhere: still a distribution
    logits[4] = low
    logits[4, 5] = 1.0                         # beside an ordinary logit it is never drawn
    logits[5, 100] = math.inf                  # the largest finite value
    logits[6, ::2] = math.nan
    for kw in (dict(), dict(temperature=0.5, top_k=20, top_p=0.9, min_p=0.01), dict(temperature=0.0)):
        tokens, logprobs = ops.sample(logits, noise, **kw)
        assert tokens[:3].tolist() == [-1, -1, 777] and (logprobs[:2] == -math.inf).all() and logprobs[2] == 0
        assert tokens[4] == 5 and tokens[5] == 100
        assert tokens[6] % 2 == 1
        _check_sample(logits[2:], noise[2:], **kw)


def test_sample_hostile_noise():
    """Noise that pulls against the ranking, NaN, zero and infinite noise."""
    V = 700
    logits = torch.linspace(5, -5, V, device=dev)[None].repeat(4, 1)
    noise = torch.exp(3 * (logits - 5))        # the least likely token wins every race
    noise[1, 3] = math.nan
    noise[2] = math.inf
    noise[3] = math.nan
    tokens, _ = ops.sample(logits, noise, top_k=torch.tensor([5, 4, 6, 6], device=dev, dtype=torch.int32))
    assert tokens.tolist() == [4, 2, 0, 0]
    zero = torch.ones(1, V, device=dev)
    zero[0, 300], zero[0, 400] = 0.0, 0.0
    assert ops.sample(logits[:1], zero)[0].item() == 300
    assert ops.sample(logits[:1], zero, top_k=50)[0].item() == 0


def test_sample_rows_have_their_own_settings_and_strides():
    B, V = 12, 9000
    g = _gen(31)
    logits, noise = torch.randn(B, V + 24, generator=g, device=dev).to(BF)[:, 11:11 + V], torch.empty(B, V + 3, device=dev).exponential_(generator=g)[:, :V]
    t = lambda *v: torch.tensor((v * B)[:B], device=dev)  # noqa: E731
    _check_sample(logits, noise, t(0.0, 0.7, 1.0, 3.0, 1.5), t(0, 1, 30, 4000).to(torch.int32), t(1.0, 0.5, 0.9), t(0.0, 0.1))


def test_sample_frequencies():
    """4096 draws of one row: each kept token's count within 5 standard deviations of its probability."""
    V, n = 40, 4096
    row = torch.randn(V, generator=_gen(2), device=dev)
    noise = torch.empty(n, V, device=dev).exponential_(generator=_gen(3))
    tokens, _ = ops.sample(row[None].repeat(n, 1), noise, top_k=8)
    p = torch.softmax(row, 0)
    kept = p.topk(8).indices
    q = torch.zeros(V, device=dev)
    q[kept] = p[kept] / p[kept].sum()
    count = torch.bincount(tokens, minlength=V).float()
    assert (count[q == 0] == 0).all()
    assert ((count - n * q).abs() <= 5 * (n * q * (1 - q)).sqrt() + 1e-6).all()


@pytest.mark.parametrize("B,V,dtype", [(1, 65537, BF), (5, 40001, F32), (37, 131073, BF), (40, 100003, F32), (150, 128257, BF)])
def test_sample_clusters_start_together(B, V, dtype):
    """Rows split over clusters of 2 to 8 CTAs whose parts differ in length, and calls one after another that leave no
    SM idle between them: a CTA is written to by its cluster only once it runs, so every call gives the same."""
    logits, noise = _logits(B, V, dtype, seed=V)
    tokens = _check_sample(logits, noise, temperature=0.8, top_k=50, top_p=0.9)
    again = [ops.sample(logits, noise, temperature=0.8, top_k=50, top_p=0.9) for _ in range(40)]
    assert all(torch.equal(t, tokens) and torch.equal(lp, again[0][1]) for t, lp in again)


@pytest.mark.parametrize("V,dtype", [(409592, F32), (409605, F32), (819184, BF), (819211, BF)])
def test_sample_rows_past_shared_memory(V, dtype):
    """Eight CTAs keep 200 KB of a row each; a longer one (the second of each pair) is read again in every pass."""
    logits, noise = _logits(2, V + 3, dtype, seed=V)
    for at in (0, 3):  # a row that starts on a 16-byte line and one that does not
        l, q = logits[:, at:at + V], noise[:, at:at + V]
        for kw in (dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=40), dict(top_p=0.8, temperature=2.0),
                   dict(min_p=0.1), dict(temperature=1.3, top_k=1000, top_p=0.95, min_p=0.001)):
            _check_sample(l, q, **kw)
    logits[0, V // 2:] = -math.inf
    logits[1] = -math.inf
    logits[1, V - 2] = 3.0
    _check_sample(logits, noise, top_p=0.9)
    assert ops.sample(logits, noise)[0][1] == V - 2


def test_sample_refusals():
    logits, noise = _logits(3, 100, BF, seed=1)

    def refused(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            ops.sample(*args, **kw)

    refused("noise must", logits, noise[:2])
    refused("noise must", logits, noise.to(BF))
    refused("logits must", logits[0], noise)
    refused("expected bf16 or fp32", logits.half(), noise)
    refused("top_p must", logits, noise, top_p=torch.ones(2, device=dev))
    refused("unit c", logits.t().contiguous().t(), noise)
    assert ops.sample(logits[:0], noise[:0])[0].shape == (0,)
