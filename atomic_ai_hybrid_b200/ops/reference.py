"""Plain-PyTorch restatements of the reference's numerical kernels.

These are the oracles every CUDA kernel of this package is tested against, and
they are also the op implementations of the unfused eager baseline model.  They
are written from the mathematics the reference states, in PyTorch:

* GDN-2 gated delta rule with per-channel decay/erase/write gates --
  token-serial ground truth (reference `atomic_ops/gdn2_wy_reference.py:33-56`)
  and the chunked WY form with the reference's clip/nan guards
  (`atomic_ops/gdn2_wy_reference.py:59-152`).
* Mamba2 SSD with per-channel ``dt`` and per-head ``A`` -- chunked form with the
  reference's clip discipline (`atomic_ops/mamba2_ssd_reference.py:56-179`) and a
  token-serial ground truth.

Shapes follow the reference: sequence tensors are ``(B, L, H, D)``.
All arithmetic is done in fp32 (or fp64 when the inputs are fp64).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F

Tensor = torch.Tensor


def sanitize(x: Tensor, clip: float) -> Tensor:
    """``nan_to_num(clip(x, -c, c))`` -- the reference's guard at kernel boundaries."""
    return torch.nan_to_num(x.clamp(-clip, clip), nan=0.0, posinf=clip, neginf=-clip)


def _nan_guard(x: Tensor, big: float = 1e4) -> Tensor:
    return torch.nan_to_num(x, nan=0.0, posinf=big, neginf=-big)


def _acc_dtype(t: Tensor) -> torch.dtype:
    return torch.float64 if t.dtype == torch.float64 else torch.float32


# --------------------------------------------------------------------------
# GDN-2
# --------------------------------------------------------------------------
def gdn2_token_serial(q, k, v, g, b, w, scale: float = 1.0, h0: Optional[Tensor] = None):
    """Token-serial GDN-2 recurrence (ground truth).

    For every token: ``h <- diag(e^g) h``; ``v' = w*v - (b*k)^T h``;
    ``h += k v'^T``; ``o = h^T (q*scale)``.  ``g`` is the per-channel log-decay.
    Returns ``(o, h_final)`` with ``o`` in the dtype of ``q`` and ``h`` fp32/fp64.
    """
    B, L, H, D = q.shape
    Dv = v.shape[-1]
    acc = _acc_dtype(q)
    h = torch.zeros(B, H, D, Dv, dtype=acc, device=q.device) if h0 is None else h0.to(acc).clone()
    alpha = torch.exp(g.to(acc))
    outs = []
    for t in range(L):
        h = h * alpha[:, t, :, :, None]
        bk = (b[:, t] * k[:, t]).to(acc)
        erase = torch.einsum("bhd,bhdv->bhv", bk, h)
        v_new = (w[:, t] * v[:, t]).to(acc) - erase
        h = h + torch.einsum("bhd,bhv->bhdv", k[:, t].to(acc), v_new)
        outs.append(torch.einsum("bhdv,bhd->bhv", h, (q[:, t] * scale).to(acc)))
    return torch.stack(outs, 1).to(q.dtype), h


def gdn2_chunk_prepare(q_c, k_c, v_c, g_c, b_c, w_c, scale: float):
    """Intra-chunk quantities of the WY form for one chunk ``(B, C, H, D)``.

    Returns ``Aqk (B,H,C,C)``, ``w_pseudo (B,C,H,D)``, ``u (B,C,H,Dv)``,
    ``kg``, ``qg`` ``(B,C,H,D)`` and ``gc_last (B,H,D)``.  ``A = (I+Akk)^-1`` is
    taken with a batched triangular solve (same matrix the reference builds with
    its row recursion, reference `atomic_ops/gdn2_wy_reference.py:18-30`).
    """
    acc = _acc_dtype(q_c)
    C = q_c.shape[1]
    gc = torch.cumsum(g_c.to(acc), dim=1)                     # (B,C,H,D)
    gcb = gc.permute(0, 2, 1, 3)                               # (B,H,C,D)
    ediff = torch.exp((gcb[:, :, :, None, :] - gcb[:, :, None, :, :]).clamp(-20.0, 20.0))
    qb = q_c.permute(0, 2, 1, 3).to(acc)
    kb = k_c.permute(0, 2, 1, 3).to(acc)
    bb = b_c.permute(0, 2, 1, 3).to(acc)
    causal = torch.tril(torch.ones(C, C, dtype=acc, device=q_c.device))
    strict = torch.tril(torch.ones(C, C, dtype=acc, device=q_c.device), -1)
    Aqk = scale * torch.einsum("bhid,bhijd,bhjd->bhij", qb, ediff, kb) * causal
    Akk = torch.einsum("bhid,bhijd,bhjd->bhij", bb * kb, ediff, kb) * strict
    Aqk = _nan_guard(Aqk)
    Akk = _nan_guard(Akk)
    eye = torch.eye(C, dtype=acc, device=q_c.device).expand_as(Akk)
    A = torch.linalg.solve_triangular(eye + Akk, eye, upper=False, unitriangular=True)
    A = _nan_guard(A)
    kb_dec = (b_c.to(acc) * k_c.to(acc)) * torch.exp(gc)
    w_pseudo = _nan_guard(torch.einsum("bhij,bjhd->bihd", A, kb_dec))
    u = _nan_guard(torch.einsum("bhij,bjhv->bihv", A, (w_c * v_c).to(acc)))
    gc_last = gc[:, -1]
    kg = k_c.to(acc) * torch.exp(gc_last[:, None] - gc)
    qg = q_c.to(acc) * torch.exp(gc)
    return Aqk, w_pseudo, u, kg, qg, gc_last


def gdn2_chunk_step(h, Aqk, w_pseudo, u, kg, qg, gc_last, scale: float):
    """Inter-chunk step of the WY form: returns ``(h_next, o_chunk, v_new)``."""
    v_new = u - torch.einsum("bihd,bhdv->bihv", w_pseudo, h)
    qh = torch.einsum("bihd,bhdv->bihv", qg, h)
    intra = torch.einsum("bhij,bjhv->bihv", Aqk, v_new)
    o = _nan_guard(scale * qh + intra)
    write = torch.einsum("bihd,bihv->bhdv", kg, v_new)
    h_new = h * torch.exp(gc_last)[..., None] + write
    h_new = sanitize(h_new, 1e4)
    return h_new, o, v_new


def gdn2_chunked(q, k, v, g, b, w, scale: float = 1.0, chunk_size: int = 64,
                 h0: Optional[Tensor] = None, checkpoint_chunks: bool = False):
    """Chunked WY GDN-2 (reference `gdn2_chunked_wy_reference`).  Differentiable."""
    B, L, H, D = q.shape
    Dv = v.shape[-1]
    assert L % chunk_size == 0, f"seq_len={L} must be divisible by chunk_size={chunk_size}"
    acc = _acc_dtype(q)
    h = torch.zeros(B, H, D, Dv, dtype=acc, device=q.device) if h0 is None else h0.to(acc)

    def one(h, qc, kc, vc, gcn, bc, wc):
        prep = gdn2_chunk_prepare(qc, kc, vc, gcn, bc, wc, scale)
        h2, o, _ = gdn2_chunk_step(h, *prep, scale)
        return h2, o

    outs = []
    for s in range(0, L, chunk_size):
        sl = slice(s, s + chunk_size)
        args = (h, q[:, sl], k[:, sl], v[:, sl], g[:, sl], b[:, sl], w[:, sl])
        if checkpoint_chunks and torch.is_grad_enabled():
            import torch.utils.checkpoint as ckpt
            h, o = ckpt.checkpoint(one, *args, use_reentrant=False)
        else:
            h, o = one(*args)
        outs.append(o)
    return torch.cat(outs, 1).to(q.dtype), h


# --------------------------------------------------------------------------
# Mamba2 SSD
# --------------------------------------------------------------------------
def ssd_token_serial(dt, A, Bm, Cm, x, state0: Optional[Tensor] = None):
    """Token-serial SSD: ``s_t = e^{dt_t A} s_{t-1} + (dt_t x_t) B_t^T``; ``y_t = s_t C_t``.

    ``dt, x: (B,L,H,P)``, ``A: (H,)``, ``B, C: (B,L,N)``.  State is ``(B,H,P,N)``.
    """
    Bsz, L, H, P = dt.shape
    N = Bm.shape[-1]
    acc = _acc_dtype(dt)
    s = torch.zeros(Bsz, H, P, N, dtype=acc, device=dt.device) if state0 is None else state0.to(acc).clone()
    Af = A.to(acc)
    ys = []
    for t in range(L):
        dA = (dt[:, t].to(acc) * Af[None, :, None]).clamp(-20.0, 20.0)
        s = s * torch.exp(dA)[..., None] + torch.einsum("bhp,bn->bhpn", dt[:, t].to(acc) * x[:, t].to(acc), Bm[:, t].to(acc))
        ys.append(torch.einsum("bhpn,bn->bhp", s, Cm[:, t].to(acc)))
    return torch.stack(ys, 1).to(x.dtype), s


def ssd_chunk(dt_c, A, B_c, C_c, x_c, state_prev):
    """One chunk of the reference SSD with its exact clip discipline
    (reference `atomic_ops/mamba2_ssd_reference.py:56-148`)."""
    acc = state_prev.dtype
    Cs = dt_c.shape[1]
    dA = sanitize(dt_c.to(acc) * A.to(acc)[None, None, :, None], 20.0)
    cum = sanitize(torch.cumsum(dA, dim=1), 1e4)                           # (b,C,h,p)
    diff = cum[:, :, None] - cum[:, None, :]                                 # (b,i,j,h,p)
    causal = torch.tril(torch.ones(Cs, Cs, dtype=acc, device=dt_c.device))[None, :, :, None, None]
    Lm = sanitize(torch.exp(diff.clamp(-20.0, 20.0)) * causal, 1e6)
    CB = sanitize(torch.einsum("bis,bjs->bij", C_c.to(acc), B_c.to(acc)), 1e4)
    dBx = sanitize(dt_c.to(acc) * x_c.to(acc), 1e4)
    y_diag = sanitize(torch.einsum("bijhp,bij,bjhp->bihp", Lm, CB, dBx), 1e4)
    dte = sanitize(torch.exp((cum[:, -1:] - cum).clamp(-20.0, 20.0)), 1e6)
    state_end = sanitize(torch.einsum("bcs,bchp->bhps", B_c.to(acc), dBx * dte), 1e4)
    decay_h = torch.exp(cum.clamp(-20.0, 0.0))
    y_off = sanitize(torch.einsum("bis,bhps->bihp", C_c.to(acc), state_prev) * decay_h, 1e4)
    dce = torch.exp(cum[:, -1].clamp(-20.0, 0.0))
    state_new = sanitize(state_prev * dce[..., None] + state_end, 1e4)
    return sanitize(y_diag + y_off, 1e4), state_new


def ssd_chunked(dt, A, Bm, Cm, x, chunk_size: int = 64, state0: Optional[Tensor] = None,
                checkpoint_chunks: bool = False):
    """Chunked SSD (reference `mamba2_ssd_reference`).  Differentiable."""
    Bsz, L, H, P = dt.shape
    N = Bm.shape[-1]
    assert L % chunk_size == 0
    acc = _acc_dtype(dt)
    s = torch.zeros(Bsz, H, P, N, dtype=acc, device=dt.device) if state0 is None else state0.to(acc)
    ys = []
    for st in range(0, L, chunk_size):
        sl = slice(st, st + chunk_size)
        args = (dt[:, sl], A, Bm[:, sl], Cm[:, sl], x[:, sl], s)
        if checkpoint_chunks and torch.is_grad_enabled():
            import torch.utils.checkpoint as ckpt
            y, s = ckpt.checkpoint(ssd_chunk, *args, use_reentrant=False)
        else:
            y, s = ssd_chunk(*args)
        ys.append(y)
    return torch.cat(ys, 1).to(x.dtype), s


# --------------------------------------------------------------------------
# Small ops
# --------------------------------------------------------------------------
def rmsnorm(x: Tensor, scale: Tensor, eps: float = 1e-6) -> Tensor:
    """Flax ``nn.RMSNorm``: fp32 statistics, ``x * rsqrt(mean(x^2)+eps) * scale``."""
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * scale.float()
    return y.to(x.dtype)


def causal_conv1d(x: Tensor, w: Tensor, bias: Optional[Tensor], silu: bool) -> Tensor:
    """Depthwise causal conv over time.  ``x (B,L,C)``, ``w (C,W)`` (flax layout
    ``(features, width)``, tap ``W-1`` hits the current token), ``bias (C,)``."""
    Bsz, L, Cn = x.shape
    W = w.shape[1]
    xt = F.pad(x.transpose(1, 2), (W - 1, 0))
    y = F.conv1d(xt, w.to(x.dtype)[:, None, :], None, groups=Cn).transpose(1, 2)
    if bias is not None:
        y = y + bias.to(x.dtype)
    return F.silu(y) if silu else y


def gelu_tanh(x: Tensor) -> Tensor:
    """``jax.nn.gelu`` default (tanh approximation)."""
    return F.gelu(x, approximate="tanh")


def safe_l2norm(x: Tensor, eps2: float) -> Tensor:
    xf = x.float()
    return (xf * torch.rsqrt((xf * xf).sum(-1, keepdim=True) + eps2)).to(x.dtype)


def label_smoothed_ce(logits: Tensor, labels: Tensor, label_smoothing: float) -> Tuple[Tensor, Tensor]:
    """Reference chunk CE (reference `optimizer.py:244-281`): returns (sum_loss, sum_mask).

    ``loss = nll*(sp - sn) - sn*sum(log_probs)`` with ``sp = 1-ls`` and
    ``sn = ls/(V-1)``; labels ``-100`` are masked out.
    """
    V = logits.shape[-1]
    lf = logits.float()
    lf = torch.nan_to_num(lf, nan=0.0, posinf=1e4, neginf=-1e4).clamp(-1e4, 1e4)
    logp = torch.log_softmax(lf, -1)
    safe = labels.clamp(0, V - 1)
    nll = -logp.gather(-1, safe[:, None].long()).squeeze(-1)
    if label_smoothing > 0:
        sp, sn = 1.0 - label_smoothing, label_smoothing / (V - 1)
        loss = nll * (sp - sn) - sn * logp.sum(-1)
    else:
        loss = nll
    mask = (labels != -100).float()
    return torch.where(mask > 0, loss, torch.zeros_like(loss)).sum(), mask.sum()


def rope_cos_sin(seq_len: int, dim: int, device=None, dtype=torch.float32):
    inv = 1.0 / (10000 ** (torch.arange(0, dim, 2, device=device, dtype=torch.float32)[: dim // 2] / dim))
    t = torch.arange(seq_len, device=device, dtype=torch.float32)
    fr = torch.outer(t, inv)
    emb = torch.cat([fr, fr], -1)
    return emb.cos().to(dtype), emb.sin().to(dtype)


def apply_rope(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    d = x.shape[-1]
    x1, x2 = x[..., : d // 2], x[..., d // 2:]
    rot = torch.cat([-x2, x1], -1)
    return x * cos.to(x.dtype) + rot * sin.to(x.dtype)


def causal_attention(q: Tensor, k: Tensor, v: Tensor, sm_scale: float) -> Tensor:
    """``(B,H,L,D)`` causal softmax attention in fp32."""
    s = torch.einsum("bhqd,bhkd->bhqk", q.float(), k.float()) * sm_scale
    L = q.shape[2]
    mask = torch.ones(L, L, dtype=torch.bool, device=q.device).tril()
    s = s.masked_fill(~mask, -1e9)
    return torch.einsum("bhqk,bhkd->bhqd", s.softmax(-1), v.float()).to(q.dtype)


def grouped_ffn(x_sorted: Tensor, group_sizes, w1: Tensor, w2: Tensor, w3: Optional[Tensor], act: str):
    """Per-expert FFN over token rows sorted by expert.  ``w1 (E,d,F)``, ``w2 (E,F,d)``,
    ``w3 (E,d,F)`` for SwiGLU.  Rows of expert ``e`` are contiguous."""
    outs = []
    start = 0
    sizes = [int(s) for s in group_sizes]
    for e, n in enumerate(sizes):
        xe = x_sorted[start:start + n]
        h = sanitize(xe @ w1[e], 1e3)
        if act == "swiglu":
            h = F.silu(h) * sanitize(xe @ w3[e], 1e3)
        else:
            h = gelu_tanh(h)
        outs.append(sanitize(h @ w2[e], 1e3))
        start += n
    return torch.cat(outs, 0) if outs else x_sorted.new_zeros(0, w2.shape[-1])


# --------------------------------------------------------------------------
# Serving: state carried between calls (updated in place)
# --------------------------------------------------------------------------
def check_no_offsets(cu_seqlens) -> None:
    if cu_seqlens is not None:
        raise ValueError("cu_seqlens packs (T, channels) rows; (B, L, channels) tokens have none")


def _sequences(x: Tensor, cu_seqlens, slots, n_slots: int):
    """``[(slot, start, end)]`` of the sequences in the flattened rows of ``x``; slot -1 is padding."""
    if x.dim() == 3:
        check_no_offsets(cu_seqlens)
        cu = [i * x.shape[1] for i in range(x.shape[0] + 1)]
    elif cu_seqlens is not None:
        T = x.shape[0]
        cu = [min(max(c, 0), T) for c in cu_seqlens.tolist()]
    else:
        cu = list(range(x.shape[0] + 1))
    which = list(range(len(cu) - 1)) if slots is None else slots.tolist()
    if len(which) != len(cu) - 1:
        raise ValueError(f"{len(cu) - 1} sequences, {len(which)} slots")
    if slots is None and len(which) > n_slots:
        raise ValueError(f"{len(which)} sequences need a state slot each, the state has {n_slots}")
    return [(s if 0 <= s < n_slots else -1, a, max(a, e)) for s, a, e in zip(which, cu[:-1], cu[1:])]


def _window_conv(x: Tensor, window: Tensor, w: Tensor, b: Optional[Tensor], acc):
    """SiLU of the causal convolution of one sequence ``(l, C)`` after ``window (3, C)``; the new window."""
    ext = torch.cat([window, x], 0)
    l = x.shape[0]
    y = sum(ext[j:j + l].to(acc) * w[:, j].to(acc) for j in range(4))
    return F.silu(y if b is None else y + b.to(acc)), ext[l:]


@torch.no_grad()
def selective_scan(x, dt, A, Bm, Cm, conv_w, conv_b, conv_state, state, cu_seqlens=None, slots=None,
                   dt_min: float = 1e-2, dt_max: float = 1.0):
    """Token-serial form of ``ops.selective_scan`` (the states are kept in ``state``'s dtype)."""
    S, H, P, N = state.shape
    C = H * P
    acc = _acc_dtype(state)
    flat = lambda t, n: t.reshape(-1, n)  # noqa: E731
    xf, dtf, Bf, Cf = flat(x, C), flat(dt, C), flat(Bm, N), flat(Cm, N)
    y = torch.zeros(xf.shape, dtype=x.dtype, device=x.device)
    a_chan = A.to(acc).repeat_interleave(P)
    for slot, s, e in _sequences(x, cu_seqlens, slots, S):
        if slot < 0 or e == s:
            continue
        xc, window = _window_conv(xf[s:e], conv_state[slot], conv_w, conv_b, acc)
        conv_state[slot] = window
        step = torch.nan_to_num(F.softplus(dtf[s:e].to(acc)).clamp(dt_min, dt_max), nan=0.0)
        a = torch.exp((step * a_chan).clamp(min=-20.0))
        u = step * sanitize(xc, 1e3)
        Bs, Cs = sanitize(Bf[s:e].to(acc), 1e3), sanitize(Cf[s:e].to(acc), 1e3)
        h = state[slot].to(acc).view(C, N)
        for t in range(e - s):
            h = h * a[t][:, None] + u[t][:, None] * Bs[t]
            y[s + t] = (h @ Cs[t]).to(y.dtype)
        state[slot] = h.view(H, P, N)
    return y.view(x.shape)


@torch.no_grad()
def gdn2_recurrent(q, k, v, b, w, f, conv_w, conv_b, decay_a, conv_state, state, cu_seqlens=None, slots=None):
    """Token-serial form of ``ops.gdn2_recurrent``."""
    S, H, D, _ = state.shape
    d = H * D
    acc = _acc_dtype(state)
    rows = [t.reshape(-1, d) for t in (q, k, v, b, w, f)]
    o = torch.zeros(rows[0].shape, dtype=q.dtype, device=q.device)
    rate = torch.exp(decay_a.to(acc).clamp(-20.0, 20.0))[:, None]
    for slot, s, e in _sequences(q, cu_seqlens, slots, S):
        if slot < 0 or e == s:
            continue
        qkv = []
        for m in range(3):
            y, conv_state[slot, m] = _window_conv(rows[m][s:e], conv_state[slot, m], conv_w[m], conv_b[m], acc)
            qkv.append(y.view(-1, H, D))
        qs, ks = (sanitize(t * torch.rsqrt((t * t).sum(-1, keepdim=True) + 1e-12), 1e3) for t in qkv[:2])
        vs = sanitize(qkv[2], 50.0)
        erase, write = (sanitize(torch.sigmoid(t[s:e].to(acc)), 1.0).view(-1, H, D) for t in rows[3:5])
        g = torch.nan_to_num(-rate * F.softplus(rows[5][s:e].to(acc)).view(-1, H, D), nan=0.0).clamp(min=-1e3)
        h = state[slot].to(acc)
        for t in range(e - s):
            h = h * torch.exp(g[t])[..., None]
            new = write[t] * vs[t] - torch.einsum("hk,hkv->hv", erase[t] * ks[t], h)
            h = h + ks[t][..., None] * new[:, None]
            o[s + t] = torch.einsum("hk,hkv->hv", qs[t], h).reshape(d).to(o.dtype)
        state[slot] = h
    return o.view(q.shape)


@torch.no_grad()
def sample(logits, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``ops.sample`` by sorting each row."""
    B, V = logits.shape
    acc = _acc_dtype(logits)

    def setting(t, dtype):
        t = t if isinstance(t, torch.Tensor) else torch.full((B,), t)
        return t.to(device=logits.device, dtype=dtype)[:, None]

    l = logits.to(acc)
    l = torch.where(torch.isnan(l), -math.inf, l).clamp(max=torch.finfo(torch.float32).max)
    T, k = setting(temperature, acc), setting(top_k, torch.long)
    greedy = ~(T > 0)
    k = torch.where(greedy, 1, torch.where(k <= 0, V, k))
    T = torch.where(greedy, 1.0, T)
    ranked, index = torch.sort(l, dim=1, descending=True, stable=True)
    top = ranked[:, :1]
    empty = top == -math.inf
    nd = torch.where(empty, -math.inf, (ranked - top) / T)  # -d
    mass = torch.exp(nd)
    before = torch.cumsum(mass, 1) - mass
    total = mass.sum(1, keepdim=True)
    rank = torch.arange(V, device=l.device)[None]
    first = rank == 0
    kept = (rank < k) & (first | (before < setting(top_p, acc) * total)) & (first | (mass >= setting(min_p, acc)))
    kept &= ranked > -math.inf
    score = nd - torch.log(noise.to(acc).gather(1, index))
    score = torch.where(kept, torch.nan_to_num(score, nan=-math.inf, posinf=math.inf, neginf=-math.inf), -math.inf)
    best = score.max(1, keepdim=True).values
    tokens = torch.where(kept & (score == best), index, V).min(1, keepdim=True).values
    tokens = torch.where(empty, -1, torch.where(best > -math.inf, tokens, index[:, :1]))
    logp = (l.gather(1, tokens.clamp(min=0)) - top) / T - torch.log(total)
    return tokens[:, 0], torch.where(empty, -math.inf, logp)[:, 0].to(torch.float64 if acc == torch.float64 else torch.float32)


@torch.no_grad()
def cached_attention(q, k, v, k_cache, v_cache, lengths, cos=None, sin=None, cu_seqlens=None, slots=None, prefix=None,
                     seen=None, mass=None, held=None, sm_scale=None):
    """``ops.cached_attention`` sequence by sequence (float64 caches compute in float64, others in fp32)."""
    S, Hk, M, D = k_cache.shape
    acc = _acc_dtype(k_cache)
    qf, kf, vf = q.reshape(-1, q.shape[-1] // D, D), k.reshape(-1, Hk, D), v.reshape(-1, Hk, D)
    H = qf.shape[1]
    if H % Hk:
        raise ValueError(f"{H} query heads do not share {Hk} key heads evenly")
    G, scale = H // Hk, 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    o = torch.zeros(qf.shape, dtype=q.dtype, device=q.device)
    rows = lengths.tolist()
    at = None if seen is None else seen.tolist()
    shared = None if prefix is None else prefix.tolist()
    for i, (slot, s, e) in enumerate(_sequences(q, cu_seqlens, slots, S)):
        n = e - s
        if slot < 0 or n == 0 or not 0 <= rows[slot] <= M - n:
            continue
        pre = -1 if shared is None else shared[i]
        if not (0 <= pre < S and 0 < rows[pre] <= M):
            pre = -1
        first, have = rows[slot], rows[slot] + n
        pos = at[slot] if at is not None else first + (rows[pre] if pre >= 0 else 0)
        if pos < 0 or (cos is not None and pos > cos.shape[0] - n):
            continue
        turn = (lambda t: t) if cos is None else (  # noqa: E731
            lambda t: apply_rope(t, cos[pos:pos + n, None].to(acc), sin[pos:pos + n, None].to(acc)))
        qs = sanitize(turn(qf[s:e].to(acc)), 1e3)
        k_cache[slot, :, first:have] = sanitize(turn(kf[s:e].to(acc)), 1e3).to(k_cache.dtype).transpose(0, 1)
        v_cache[slot, :, first:have] = sanitize(vf[s:e].to(acc), 1e3).to(v_cache.dtype).transpose(0, 1)
        keys, values = k_cache[slot, :, :have], v_cache[slot, :, :have]
        if pre >= 0:
            keys = torch.cat([k_cache[pre, :, :rows[pre]], keys], 1)
            values = torch.cat([v_cache[pre, :, :rows[pre]], values], 1)
        w = torch.einsum("tkgd,kjd->kgtj", qs.view(n, Hk, G, D), keys.to(acc)) * scale
        hidden = torch.ones(n, keys.shape[1], dtype=torch.bool, device=q.device).triu(keys.shape[1] - n + 1)
        w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
        o[s:e] = torch.einsum("kgtj,kjd->tkgd", w, values.to(acc)).reshape(n, H, D).to(o.dtype)
        if mass is not None:
            mass[slot, :, first:have] = 0
            mass[slot, :, :have] += w.sum((1, 2))[:, keys.shape[1] - have:].to(mass.dtype)
            held[slot, :, first:have] = torch.arange(pos, pos + n, dtype=held.dtype, device=held.device)
    return o.view(q.shape)


@torch.no_grad()
def cache_evict(k_cache, v_cache, mass, held, lengths, seen, keep, recent=0, slots=None):
    """``ops.cache_evict`` head by head."""
    S, Hk, M, _ = k_cache.shape
    rows, at = lengths.tolist(), seen.tolist()
    for slot in range(S) if slots is None else dict.fromkeys(slots.tolist()):
        if not 0 <= slot < S or not keep < rows[slot] <= M:
            continue
        n = rows[slot]
        gathered = mass[slot, :, :n]
        low = torch.isnan(gathered) | (gathered == -math.inf)
        newest = held[slot, :, :n].long() >= at[slot] - recent
        order = torch.sort(torch.where(newest | low, -math.inf, gathered), dim=-1, descending=True, stable=True).indices
        order = order.gather(1, torch.sort(newest.gather(1, order).int(), dim=-1, descending=True, stable=True).indices)
        kept = torch.zeros_like(newest).scatter_(-1, order[:, :keep], True)
        h, hole = torch.nonzero(~kept[:, :keep], as_tuple=True)
        row = torch.nonzero(kept[:, keep:], as_tuple=True)[1] + keep
        for t in (k_cache, v_cache, mass, held):
            t[slot, h, hole] = t[slot, h, row]


def _score_rows(logits, temperature):
    """Scores below their row's largest, and the rows in which there is one."""
    x = torch.where(torch.isnan(logits), -math.inf, logits).clamp(max=torch.finfo(torch.float32).max)
    top = x.max(1, keepdim=True).values
    some = top > -math.inf
    return (x - torch.where(some, top, 0.0)) / temperature, some


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature):
        ctx.save_for_backward(logits, tokens)
        ctx.temperature = temperature
        d, some = _score_rows(logits.to(_acc_dtype(logits)), temperature)
        p = torch.exp(d)
        total = p.sum(1, keepdim=True)
        logp = torch.where(some, d - torch.log(total), -math.inf)
        given = (tokens >= 0) & (tokens < logits.shape[1])
        lp = torch.where(given, logp.gather(1, torch.where(given, tokens, 0)[:, None])[:, 0], 0.0)
        entropy = -torch.where(p > 0, p / total * logp, 0.0).sum(1)
        return lp, entropy

    @staticmethod
    def backward(ctx, g, ge):
        logits, tokens = ctx.saved_tensors
        d, some = _score_rows(logits.to(_acc_dtype(logits)), ctx.temperature)
        p = torch.exp(d)
        total = p.sum(1, keepdim=True)
        p, logp = p / total, torch.where(p > 0, d - torch.log(total), 0.0)
        entropy = -(p * logp).sum(1, keepdim=True)
        given = (tokens >= 0) & (tokens < logits.shape[1])
        g = torch.where(given, g, 0.0)[:, None].to(p.dtype)
        dx = -p * (g + ge[:, None].to(p.dtype) * (logp + entropy))
        dx.scatter_add_(1, torch.where(given, tokens, 0)[:, None], g)
        # tokens without probability stay without gradient, the given one among them
        dx = torch.where((d > -math.inf) & some, dx, 0.0) / ctx.temperature
        return dx.to(logits.dtype), None, None


def token_logprobs(logits, tokens, top: int = 0, temperature: float = 1.0):
    """``ops.token_logprobs`` from whole rows (the alternatives by sorting)."""
    lp, entropy = _TokenLogprobs.apply(logits, tokens, temperature)
    if not top:
        return lp, entropy
    with torch.no_grad():
        d, some = _score_rows(logits.to(_acc_dtype(logits)), temperature)
        best, index = torch.sort(d, dim=1, descending=True, stable=True)
        best, index = best[:, :top], index[:, :top]
        best = torch.where(some, best - torch.log(torch.exp(d).sum(1, keepdim=True)), -math.inf)
        index = torch.where(best > -math.inf, index, -1)
    return lp, entropy, index, best


def newton_schulz3(g: Tensor, steps: int = 3, eps: float = 1e-4) -> Tensor:
    """Reference Muon orthogonalisation (reference `optimizer.py:53-77`)."""
    if g.ndim == 3:
        nrm = torch.linalg.vector_norm(g, dim=(-2, -1), keepdim=True)
        nrm = torch.where(nrm < eps, torch.ones_like(nrm), nrm)
        X = g / nrm
        for _ in range(steps):
            X = 1.5 * X - 0.5 * (X @ X.transpose(-1, -2) @ X)
            X = torch.nan_to_num(X, nan=0.0, posinf=0.0, neginf=0.0)
    else:
        nrm = torch.linalg.vector_norm(g)
        nrm = torch.where(nrm < eps, torch.ones_like(nrm), nrm)
        X = g / nrm
        for _ in range(steps):
            X = 1.5 * X - 0.5 * (X @ X.T @ X)
            X = torch.nan_to_num(X, nan=0.0, posinf=0.0, neginf=0.0)
    return X


def flops_gdn_chunked(B: int, L: int, H: int, D: int, C: int) -> float:
    """Matmul FLOPs of one chunked GDN forward (used for scan TFLOP/s)."""
    nc = L // C
    per_chunk = (2 * C * C * D * 2            # Aqk, Akk
                 + 2 * C * C * D * 2          # w_pseudo, u
                 + 2 * C * D * D * 3          # w h, q h, k^T v
                 + 2 * C * C * D)             # Aqk v_new
    return float(B * H * nc * per_chunk)


def flops_ssd_chunked(B: int, L: int, H: int, P: int, N: int, C: int) -> float:
    nc = L // C
    per_chunk = (2 * C * C * N + 2 * C * C * P      # CB, y_diag
                 + 2 * C * P * N * 2)               # state_end, y_off
    return float(B * H * nc * per_chunk)


__all__ = [n for n in dir() if not n.startswith("_")]
_ = math
