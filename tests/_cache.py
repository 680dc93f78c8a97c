"""Inputs and 64-bit definitions that the tests of the cache operators share, on the CPU and on the GPU."""
import math

import torch

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def gen(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def offsets(lens, device):
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens, dtype=torch.int32), 0)
    return cu.to(device)


def tables(n, D, device):
    a = torch.arange(n, dtype=F64)[:, None] / 10000 ** (torch.arange(0, D, 2, dtype=F64) / D)
    a = torch.cat([a, a], -1)
    return a.cos().float().to(device), a.sin().float().to(device)


def attention_inputs(lens, had, H, Hk, D, dtype, device, prefix=None, tracked=False, seed=0, behind=math.nan, std=1.5, extra=3):
    """Arguments of ``cached_attention`` for sequences of ``lens`` new tokens over ``had`` rows; ``prefix``: rows of each
    distinct prefix and each sequence's choice, ``(rows, which)`` (-1: none).  The cache holds ``behind`` where no row is."""
    g = gen(seed, device)
    B, T = len(lens), sum(lens)
    rows, which = prefix if prefix else ([], [-1] * B)
    S = B + len(rows) + extra
    M = max([h + n for h, n in zip(had, lens)] + list(rows) + [1]) + 3
    order = torch.randperm(S, generator=g, device=device)
    slots, pre = order[:B], order[B:B + len(rows)]
    lengths = torch.zeros(S, dtype=torch.int32, device=device)
    lengths[slots] = torch.tensor(had, dtype=torch.int32, device=device)
    if rows:
        lengths[pre] = torch.tensor(rows, dtype=torch.int32, device=device)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    has = torch.arange(M, device=device) < lengths[:, None]
    caches = [torch.where(has[:, None, :, None], r(S, Hk, M, D), behind).to(dtype) for _ in range(2)]
    a = dict(q=(r(T, H * D) * std).to(dtype), k=r(T, Hk * D).to(dtype), v=r(T, Hk * D).to(dtype), k_cache=caches[0],
             v_cache=caches[1], lengths=lengths, cu_seqlens=offsets(lens, device), slots=slots.to(torch.int32))
    a["cos"], a["sin"] = tables(M + max(rows, default=0) + 1, D, device)
    if prefix:
        a["prefix"] = torch.tensor([int(pre[w]) if w >= 0 else -1 for w in which], dtype=torch.int32, device=device)
    if tracked:
        a["mass"] = torch.where(has[:, None], torch.rand(S, Hk, M, generator=g, device=device) * 3, 0.5)
        a["held"] = torch.where(has[:, None], torch.arange(M, device=device, dtype=torch.int32), -7).expand(S, Hk, M).contiguous()
    return a


def copied(a):
    return {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in a.items()}


def attention_truth(q, k, v, k_cache, v_cache, lengths, cos=None, sin=None, cu_seqlens=None, slots=None, prefix=None, seen=None,
                    mass=None, held=None, sm_scale=None):
    """``ops.cached_attention`` row by row in 64 bits.  Returns ``(o, bound, caches, mass, held, gained)``: ``bound`` is
    what roundings of the queries and of the weights to bf16 may change in ``o``, ``gained`` what they may in ``mass``."""
    S, Hk, M, D = k_cache.shape
    T = q.shape[0]
    H = q.shape[1] // D
    G = H // Hk
    scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    kc, vc = k_cache.clone(), v_cache.clone()
    o = torch.zeros(T, H, D, dtype=F64, device=q.device)
    bound = torch.zeros(T, H, D, dtype=F64, device=q.device)
    ms, hd = (None, None) if mass is None else (mass.double(), held.clone())
    gained = None if mass is None else torch.zeros_like(ms)
    cu = cu_seqlens.tolist() if cu_seqlens is not None else list(range(T + 1))
    half = D // 2
    for i, (b, e) in enumerate(zip(cu[:-1], cu[1:])):
        slot, n = int(slots[i]) if slots is not None else i, e - b
        if not 0 <= slot < S or n <= 0 or not 0 <= int(lengths[slot]) <= M - n:
            continue
        first, pre = int(lengths[slot]), -1 if prefix is None else int(prefix[i])
        P = int(lengths[pre]) if 0 <= pre < S else 0
        if not 0 < P <= M:
            P, pre = 0, -1
        pos = int(seen[slot]) if seen is not None else first + P
        if pos < 0 or cos is not None and pos + n > cos.shape[0]:
            continue

        def turned(x, heads):
            x = x.double().view(n, heads, D)
            if cos is not None:
                c, s = (t[pos:pos + n, None, :half].double() for t in (cos, sin))
                x = torch.cat([x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s], -1)
            return x.nan_to_num(0.0, 1e3, -1e3).clamp(-1e3, 1e3)

        qs, ks = turned(q[b:e], H), turned(k[b:e], Hk)
        vs = v[b:e].double().view(n, Hk, D).nan_to_num(0.0, 1e3, -1e3).clamp(-1e3, 1e3)
        kc[slot, :, first:first + n] = ks.transpose(0, 1).to(kc.dtype)
        vc[slot, :, first:first + n] = vs.transpose(0, 1).to(vc.dtype)
        if mass is not None:
            ms[slot, :, first:first + n] = 0
            hd[slot, :, first:first + n] = torch.arange(pos, pos + n, dtype=torch.int32, device=q.device)
        for h in range(H):
            own = slice(0, first + n)
            keys, values = kc[slot, h // G, own].double(), vc[slot, h // G, own].double()
            if pre >= 0:
                keys = torch.cat([kc[pre, h // G, :P].double(), keys])
                values = torch.cat([vc[pre, h // G, :P].double(), values])
            hidden = torch.arange(P + first + n, device=q.device) > P + first + torch.arange(n, device=q.device)[:, None]
            s = (qs[:, h] @ keys.t() * scale).masked_fill(hidden, -math.inf)
            p = torch.softmax(s, -1)
            o[b:e, h] = p @ values
            # a query rounded by at most 2^-8 of each channel moves a score by d, a weight by at most e^(2 d); and each
            # weight is rounded by 2^-8 itself (bf16 rounds by half a step, finfo.eps / 2)
            d = 2.0 ** -8 * abs(scale) * (qs[:, h].abs() @ keys.abs().t()).masked_fill(hidden, 0).max(-1, keepdim=True).values
            bound[b:e, h] = (2.0 ** -8 + torch.expm1(2 * d)) * (p @ values.abs())
            if mass is not None:
                ms[slot, h // G, own] += p.sum(0)[P:]
                gained[slot, h // G, own] += (torch.expm1(2 * d) * p).sum(0)[P:]
    return o.view(T, H * D), bound.view(T, H * D), (kc, vc), ms, hd, gained


def check_attention(call, a, out_half_step):
    """Runs ``call(**a)`` on a copy and holds everything that it returns and changes to the 64-bit definition.
    ``out_half_step``: half a step of the output's type (2^-8 for bf16); fp32 arithmetic adds 1e-5 (a thousand sums of 2^-24)."""
    b = copied(a)
    y = call(**b)
    given = {n: t for n, t in a.items() if n not in ("q", "k", "v")}
    flat = {n: a[n].reshape(-1, a[n].shape[-1]) for n in ("q", "k", "v")}
    if a["q"].dim() == 3:
        given["cu_seqlens"] = offsets([a["q"].shape[1]] * a["q"].shape[0], a["q"].device)
    o, bound, caches, mass, held, gained = attention_truth(**flat, **given)
    rounded = a["k_cache"].dtype == BF
    y64 = y.reshape(o.shape).double()
    err = (y64 - o).abs()
    lim = out_half_step * o.abs() + (bound * (1 + out_half_step) if rounded else 0) + 1e-5 * (1 + o.abs())
    assert y.shape == a["q"].shape and y.dtype == a["q"].dtype
    assert (err <= lim).all(), float((err - lim).max())
    # roundings in no common direction: queries, weights and outputs, each 2^-8 / sqrt(3) on average, the queries' by the scores' spread
    if rounded and o.norm() > 0:
        assert (y64 - o).norm() <= 2.0 ** -7 * o.norm(), float((y64 - o).norm() / o.norm())
    for name, want in zip(("k_cache", "v_cache"), caches):
        got = b[name].double()
        want = want.double()
        fresh = ~(want == a[name].double()) & ~(want.isnan() & a[name].isnan())
        # a rotated key comes from two products and a sum in fp32 before it is rounded: next to a border it may round the other way
        tol = 2 * torch.finfo(a[name].dtype).eps * want.abs() + 1e-6 if name == "k_cache" else torch.zeros((), dtype=F64)
        assert (~fresh | ((got - want).abs() <= tol)).all(), name
        same = got.nan_to_num(12345.0) == a[name].double().nan_to_num(12345.0)
        assert (same | fresh).all(), f"{name}: rows that are not this call's changed"
    if mass is not None:
        assert torch.equal(b["held"], held)
        err = (b["mass"].double() - mass).abs()
        assert (err <= (gained if rounded else 0) + 1e-5 * (1 + mass.abs())).all(), float(err.max())
    for n in ("lengths", "seen", "prefix", "slots"):
        if isinstance(a.get(n), torch.Tensor):
            assert torch.equal(a[n], b[n])
    return y, b


def evict_truth(k_cache, v_cache, mass, held, lengths, seen, keep, recent=0, slots=None):
    """``ops.cache_evict`` by sorting lists of each head's rows; returns the four tensors."""
    out = [t.clone() for t in (k_cache, v_cache, mass, held)]
    S, Hk, M = mass.shape
    for slot in range(S) if slots is None else slots.tolist():
        n = int(lengths[slot]) if 0 <= slot < S else 0
        if n <= keep or n > M:
            continue
        for h in range(Hk):
            m, p = mass[slot, h, :n].tolist(), held[slot, h, :n].tolist()
            new = [x >= int(seen[slot]) - recent for x in p]
            worth = [math.inf if x == math.inf else -math.inf if math.isnan(x) else x for x in m]
            order = sorted(range(n), key=lambda i: (not new[i], 0.0 if new[i] else -worth[i], i))
            kept = set(order[:keep])
            holes = [i for i in range(keep) if i not in kept]
            rows = [i for i in range(keep, n) if i in kept]
            for t in out:
                t[slot, h, holes] = t[slot, h, rows].clone()
    return out


def score_truth(logits, tokens, top=0, temperature=1.0, g=None, ge=None):
    """``ops.token_logprobs`` and its gradient in 64 bits."""
    x = torch.where(torch.isnan(logits), -math.inf, logits.double()).clamp(max=torch.finfo(F32).max) / temperature
    some = x.max(1, keepdim=True).values > -math.inf
    logp = torch.where(some, torch.log_softmax(torch.where(some, x, 0.0), 1), -math.inf)
    p = logp.exp()
    entropy = -torch.xlogy(p, p).sum(1)
    given = (tokens >= 0) & (tokens < logits.shape[1])
    at = torch.where(given, tokens, 0)[:, None]
    lp = torch.where(given, logp.gather(1, at)[:, 0], 0.0)
    out = [lp, entropy]
    if top:
        best, index = torch.sort(x, dim=1, descending=True, stable=True)
        best = logp.gather(1, index)[:, :top]
        out += [torch.where(best > -math.inf, index[:, :top], -1), best]
    if g is not None:
        one = torch.zeros_like(p).scatter_(1, at, 1.0) * given[:, None]
        dx = g.double()[:, None] * (one - p * given[:, None]) - ge.double()[:, None] * (torch.xlogy(p, p) + p * entropy[:, None])
        out.append(torch.where(logp > -math.inf, dx, 0.0) / temperature)
    return out


def extreme_scores(dtype, device):
    """Logits with masked places, and logits near the type's largest: (logits, tokens, temperatures)."""
    x = torch.randn(4, 5003, generator=torch.Generator().manual_seed(3)) * 3
    x[0, :100] = -math.inf
    x[1, ::7] = math.nan
    x[2, 5:] = torch.finfo(dtype).min
    y = torch.tensor([4000, 4001, 3, -100])
    huge = torch.linspace(0, 2.9e38, 1000).roll(300)[None]
    return [(x.to(dtype).to(device), y.to(device), T) for T in (1e-3, 1e-9, 1e-12)] + \
        [(huge.to(dtype).to(device), y[2:3].to(device), T) for T in (1.0, 1e30, 1e37)]
