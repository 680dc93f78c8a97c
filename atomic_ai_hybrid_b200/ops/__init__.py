"""Operator entry points used by the models.

Two implementations exist for every op:

* ``"cuda"``  -- the product path: hand-written sm_100a kernels in
  ``atomic_ai_hybrid_b200/csrc`` (loaded from the in-tree extension
  ``_ahb_cuda*.so``).  Selected by default for CUDA tensors.  If the extension
  is missing on a machine with a GPU the op raises instead of falling back.
* ``"eager"`` -- plain PyTorch (``ops.reference``), the unfused baseline of the
  benchmark and the only path for CPU tensors.

``set_impl("eager")`` forces the baseline on the GPU (used by ``bench.py --impl
eager``); ``set_impl("cuda")`` is the default.
"""
from __future__ import annotations

import contextlib
import os
from typing import Optional

import torch
import torch.nn.functional as F

from . import reference as R

_IMPL = os.environ.get("AHB_IMPL", "cuda")


def set_impl(name: str) -> None:
    global _IMPL
    assert name in ("cuda", "eager"), name
    _IMPL = name


def get_impl() -> str:
    return _IMPL


@contextlib.contextmanager
def impl(name: str):
    old = _IMPL
    set_impl(name)
    try:
        yield
    finally:
        set_impl(old)


def use_cuda(*tensors: torch.Tensor) -> bool:
    """True when the CUDA kernels must run for these tensors."""
    if _IMPL != "cuda":
        return False
    return all(t.is_cuda for t in tensors if isinstance(t, torch.Tensor))


def _k():
    from . import kernels
    return kernels


# ---------------------------------------------------------------- gradient guards
class _GradSanitize(torch.autograd.Function):
    """Identity forward; backward clips the cotangent to ``+-clip`` and replaces
    non-finite values (reference ``make_grad_sanitizer``, `model.py:192-217`)."""

    @staticmethod
    def forward(ctx, x, clip, tag):
        ctx.clip, ctx.tag = clip, tag
        return x.view_as(x)

    @staticmethod
    def backward(ctx, g):
        if ctx.tag is not None:
            from ..utils.diag import DIAG
            DIAG.grad_fixed(ctx.tag, g)
        if g.is_cuda and _IMPL == "cuda":
            return _k().sanitize(g, ctx.clip), None, None
        return R.sanitize(g, ctx.clip), None, None


def grad_sanitize(x: torch.Tensor, clip: float = 1e3, tag: Optional[str] = None) -> torch.Tensor:
    """``tag``: report a non-finite incoming gradient as ``[BWD-FIX]`` (``utils.diag``)."""
    if not torch.is_grad_enabled() or not x.requires_grad:
        return x
    return _GradSanitize.apply(x, clip, tag)


def sanitize(x: torch.Tensor, clip: float) -> torch.Tensor:
    if use_cuda(x):
        return _k().sanitize_fwd(x, clip)
    return R.sanitize(x, clip)


# ---------------------------------------------------------------- dense / norm
def linear(x: torch.Tensor, kernel: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ kernel (+ bias)`` in the dtype of ``x`` (cuBLAS for plain GEMMs)."""
    w = kernel if kernel.dtype == x.dtype else kernel.to(x.dtype)
    if bias is not None:
        b = bias if bias.dtype == x.dtype else bias.to(x.dtype)
        return torch.addmm(b, x.reshape(-1, x.shape[-1]), w).view(*x.shape[:-1], w.shape[-1])
    return torch.matmul(x, w)


def rmsnorm(x: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    if use_cuda(x):
        return _k().rmsnorm(x, scale, eps)
    return R.rmsnorm(x, scale, eps)


def conv1d(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor], silu: bool = True,
           clip: Optional[float] = None) -> torch.Tensor:
    """Depthwise causal conv (+bias, +SiLU, optional output clamp)."""
    if use_cuda(x):
        return _k().conv1d(x, w, b, silu, clip)
    y = R.causal_conv1d(x, w, b, silu)
    return y.clamp(-clip, clip) if clip is not None else y


# ---------------------------------------------------------------- sequence mixers
def gdn2(q, k, v, w, b, g, scale: float = 1.0, chunk: int = 64, h0=None, return_final: bool = False):
    """GDN-2 chunked delta rule; ``(B,L,H,D)`` inputs, per-channel gates.  ``h0`` (B,H,D,D)
    is the state before the first token; ``return_final`` returns ``(o, h_final)``."""
    if use_cuda(q):
        return _k().gdn2(q, k, v, w, b, g, scale, chunk, h0=h0, return_final=return_final)
    o, hf = R.gdn2_chunked(q, k, v, g, b, w, scale, chunk, h0=h0, checkpoint_chunks=True)
    return (o, hf) if return_final else o


def ssd(dt, A, Bm, Cm, x, chunk: int = 64, state0=None, return_final: bool = False):
    """Mamba2 SSD; ``dt, x (B,L,H,P)``, ``A (H,)``, ``B, C (B,L,N)``.  ``state0`` (B,H,P,N)
    is the state before the first token; ``return_final`` returns ``(y, s_final)``."""
    if use_cuda(x):
        return _k().ssd(dt, A, Bm, Cm, x, chunk, state0=state0, return_final=return_final)
    y, sf = R.ssd_chunked(dt, A, Bm, Cm, x, chunk, state0=state0, checkpoint_chunks=True)
    return (y, sf) if return_final else y


def attention(q, k, v, sm_scale: float) -> torch.Tensor:
    """Causal attention on ``(B,H,L,D)``."""
    if use_cuda(q):
        return _k().attention(q, k, v, sm_scale)
    if q.dtype == torch.float32 or q.dtype == torch.float64:
        return R.causal_attention(q, k, v, sm_scale)
    return F.scaled_dot_product_attention(q, k, v, is_causal=True, scale=sm_scale)


# ---------------------------------------------------------------- MoE
def grouped_ffn(x_sorted, group_sizes, w1, w2, w3, act: str, group_sizes_cpu=None):
    if use_cuda(x_sorted):
        return _k().grouped_ffn(x_sorted, group_sizes, w1, w2, w3, act)
    sizes = group_sizes_cpu if group_sizes_cpu is not None else group_sizes.tolist()
    dt = x_sorted.dtype
    return R.grouped_ffn(x_sorted, sizes, w1.to(dt), w2.to(dt), None if w3 is None else w3.to(dt), act)


# ---------------------------------------------------------------- serving (state carried between calls)
def selective_scan(x, dt, A, Bm, Cm, conv_w, conv_b, conv_state, state, cu_seqlens=None, slots=None,
                   dt_min: float = 1e-2, dt_max: float = 1.0) -> torch.Tensor:
    """Mamba2's short causal convolution and scan from and into a kept state; no gradient.

    ``x`` (the scan's input before the convolution) and ``dt`` (before softplus, its bias added)
    have ``C`` channels in ``A.numel()`` heads (``A`` negative), ``Bm`` and ``Cm`` have ``N`` states::

        xc_t = clip(silu(sum_j conv_w[:, j] x_{t-3+j} + conv_b), 1e3),  dt_t = clamp(softplus(dt_t), dt_min, dt_max)
        S_t  = e^{max(dt_t A, -20)} S_{t-1} + dt_t xc_t B_t^T,          y_t = S_t C_t

    Tokens come as ``(T, C)`` rows packed by ``cu_seqlens`` (int32, ``sequences + 1`` offsets on the
    device, none below the one before; sequences of any length, also none; rows that none covers come out
    as zeros), as ``(B, L, C)``, or as ``(B, C)`` rows of one token
    each.  ``conv_state (S, 3, C)`` holds the last three rows of ``x`` in its dtype and ``state
    (S, H, P, N)`` the fp32 scan state; both are updated in place.  Sequence ``i`` owns slot
    ``slots[i]`` (int32, all different; default ``i``); one with a slot outside ``[0, S)`` is padding:
    zeros come out and no state is touched.  The state moves past every token given: to go back, as after drafted
    tokens that were not accepted, copy the slots before.  Returns ``y`` shaped like ``x``."""
    if x.is_cuda and _IMPL == "cuda":
        return _k().selective_scan(x, dt, A, Bm, Cm, conv_w, conv_b, conv_state, state, cu_seqlens, slots, dt_min,
                                   dt_max)
    return R.selective_scan(x, dt, A, Bm, Cm, conv_w, conv_b, conv_state, state, cu_seqlens, slots, dt_min, dt_max)


def gdn2_recurrent(q, k, v, b, w, f, conv_w, conv_b, decay_a, conv_state, state, cu_seqlens=None,
                   slots=None) -> torch.Tensor:
    """GDN-2 token by token from and into a kept state (single tokens and a few at once; ``gdn2``
    is the chunked form for long sequences); no gradient.

    The six inputs are the layer's projections before convolution and gates, ``d = H D`` channels
    each; ``conv_w`` / ``conv_b`` are the three convolutions of ``q, k, v``::

        q, k, v = silu(conv(.)); v clipped to 50; q, k l2-normalised per head
        h <- diag(exp(-e^decay_a softplus(f))) h;  n = sigmoid(w) v - (sigmoid(b) k)^T h
        h <- h + k n^T;  o = q^T h

    Tokens, ``cu_seqlens`` and ``slots`` as in ``selective_scan``; ``conv_state (S, 3, 3, d)`` holds
    the last three rows of ``q, k, v`` (in that order) and ``state (S, H, D, D)`` the fp32 state, both
    updated in place.  Returns ``o`` shaped like ``q``."""
    if q.is_cuda and _IMPL == "cuda":
        return _k().gdn2_recurrent(q, k, v, b, w, f, conv_w, conv_b, decay_a, conv_state, state, cu_seqlens, slots)
    return R.gdn2_recurrent(q, k, v, b, w, f, conv_w, conv_b, decay_a, conv_state, state, cu_seqlens, slots)


def sample(logits, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The next token of every row of ``logits (B, V)`` from given noise; returns ``(tokens int64,
    logprobs fp32)``.

    ``noise (B, V)`` fp32 holds Exp(1) draws (``torch.empty(B, V).exponential_()``).  The settings are
    numbers or ``(B,)`` tensors.  Tokens are ranked by (logit descending, index ascending); of the
    row's distribution ``softmax(logits / temperature)`` those are kept whose rank is below ``top_k``
    (0 or less: no limit), with less than ``top_p`` of the mass ranked before them (the first one
    always), and with at least ``min_p`` times the first one's probability.  Each rule looks at the whole tempered row:
    ``top_p`` counts the mass of tokens that ``top_k`` cuts too, where samplers that renormalise after ``top_k`` keep
    fewer tokens for the same settings.  A rule that no mass can meet (``top_p <= 0``, ``min_p > 1``, NaN) keeps the
    first token alone.  The token is the kept
    one with the largest ``log p - log noise`` (ties: lowest index), which draws from the kept ones by
    their probability (a row without any such score gives the first).  ``temperature <= 0`` takes the first token and
    tempers by 1 for ``logprobs``, the log-probability before anything is cut.  NaN and ``-inf`` logits are never drawn; a row
    of nothing else gives token -1 and ``-inf``."""
    if logits.is_cuda and _IMPL == "cuda":
        return _k().sample(logits, noise, temperature, top_k, top_p, min_p)
    return R.sample(logits, noise, temperature, top_k, top_p, min_p)


def cached_attention(q, k, v, k_cache, v_cache, lengths, cos=None, sin=None, cu_seqlens=None, slots=None, prefix=None,
                     seen=None, mass=None, held=None, sm_scale: Optional[float] = None) -> torch.Tensor:
    """Attention of new tokens over a kept cache, into which their keys and values go first; no gradient.

    ``q`` has ``H D`` channels, ``k`` and ``v`` have ``Hk D`` (query head ``h`` reads key head ``h // (H // Hk)``; at most 128 share one),
    before rotation; tokens, ``cu_seqlens`` and ``slots`` as in ``selective_scan``.  ``k_cache`` and ``v_cache``
    ``(S, Hk, M, D)`` hold ``lengths[s]`` rows (int32) of slot ``s``.  Sequence ``i`` in slot ``s``::

        q, k = rotated by the table rows cos, sin [seen[s] + t]  (fp32, one row a position, halves repeated)
        q, k, v clipped to 1e3;  row lengths[s] + t of the cache <- k_t, v_t, rounded to its type
        o_t = sum_j p_tj v_j,  p_t = softmax_j(sm_scale q_t k_j)  over the prefix's rows and own rows j <= lengths[s] + t

    Without tables nothing is rotated; ``sm_scale``, at most 1e28 either way, is ``1 / sqrt(D)`` by default.  ``prefix`` (int32, one a sequence): the
    slot whose rows the sequence sees before its own, any value outside ``[0, S)`` for none; neighbours in the batch
    with the same one read its rows once for all.  ``seen`` (int32, one a slot) is the position of a slot's next token,
    by default its rows and its prefix's.  ``mass`` (fp32) and ``held`` (int32), both ``(S, Hk, M)`` or neither: new
    rows start with mass 0 and hold their position, then every own row's mass grows by the ``p_tj`` that it got from the call's
    tokens and query heads (a prefix's rows gather none).  Scores have 32 bits: a mass is off by some 2^-22 of the size of its tokens' largest
    scores, next to nothing where these are tens or hundreds.

    ``lengths`` and ``seen`` stay as they are, for the next layer's call: the caller moves them past the tokens.  The
    cache is read below ``lengths`` only, rows that earlier calls wrote, or others within the same clip: what lies behind may be anything.  A
    sequence whose slot is outside ``[0, S)``, whose rows would not fit into ``M`` or whose positions have no table row is
    padding: zeros come out and nothing is written.  Returns ``o`` shaped like ``q``."""
    if q.is_cuda and _IMPL == "cuda":
        return _k().cached_attention(q, k, v, k_cache, v_cache, lengths, cos, sin, cu_seqlens, slots, prefix, seen, mass,
                                     held, sm_scale)
    return R.cached_attention(q, k, v, k_cache, v_cache, lengths, cos, sin, cu_seqlens, slots, prefix, seen, mass, held,
                              sm_scale)


def cache_evict(k_cache, v_cache, mass, held, lengths, seen, keep: int, recent: int = 0, slots=None) -> None:
    """Thins the cache of ``cached_attention`` out to ``keep`` rows per key head, in place; no gradient.

    Of the ``lengths[s]`` rows of every slot ``s`` in ``slots`` (int32, one given twice counts once; default all) those are kept whose
    position ``held`` is at least ``seen[s] - recent`` (``recent <= keep``: the newest ones) and then those with the largest
    ``mass``, up to ``keep`` in all (ties: the lower row; NaN and ``-inf`` last).  Kept rows below ``keep`` stay where they are; the
    others fill the rows below ``keep`` that were given up, in the order of both, with their mass and position.  What
    lies behind is left as it was.  Slots outside ``[0, S)`` and those that hold ``keep`` rows or fewer stay as they are.

    Every head keeps rows of its own.  ``lengths`` stays as it is, for the next layer's call: the caller sets it to at most ``keep``."""
    if not 0 <= recent <= keep or keep < 1:
        raise ValueError(f"cache_evict: keep must be at least 1 and recent between 0 and keep, got keep={keep}, recent={recent}")
    if k_cache.is_cuda and _IMPL == "cuda":
        return _k().cache_evict(k_cache, v_cache, mass, held, lengths, seen, keep, recent, slots)
    return R.cache_evict(k_cache, v_cache, mass, held, lengths, seen, keep, recent, slots)


MAX_ALTERNATIVES = 64


def token_logprobs(logits, tokens, top: int = 0, temperature: float = 1.0):
    """Log-probabilities of given tokens under ``p = softmax(logits / temperature)``: ``logits (R, V)``, ``tokens (R,)``
    int64; returns ``(logprobs, entropy)``, fp32 ``(R,)`` each::

        logprobs = log p[token],  entropy = -sum_v p_v log p_v
        d logits_v = (g_logprobs ([v == token] - p_v) - g_entropy p_v (log p_v + entropy)) / temperature

    with ``top`` (at most 64 and ``V``) also ``(top_tokens int64, top_logprobs fp32)``, both ``(R, top)``: the likeliest
    ones (ties: lowest index), which carry no gradient.  A token outside ``[0, V)`` (-100, say) has log-probability 0 and no
    gradient.  NaN and ``-inf`` logits have no probability, +inf counts as the largest finite number; a row of nothing else
    gives ``-inf``, entropy 0, alternatives -1 and no gradient, and so do alternatives without probability.

    To capture the backward pass into a CUDA graph, let go of earlier graphs of the same leaf first: PyTorch hands a leaf's
    gradient over on the stream of its oldest living graph, and a capture that meets another stream there fails."""
    if logits.dim() != 2 or tokens.shape != logits.shape[:1] or tokens.dtype != torch.int64:
        raise ValueError(f"token_logprobs: one int64 token for each row of logits (R, V), got {tokens.dtype} {tuple(tokens.shape)} "
                         f"for {tuple(logits.shape)}")
    if not 0 <= top <= min(MAX_ALTERNATIVES, logits.shape[1]):
        raise ValueError(f"token_logprobs: top must lie between 0 and {min(MAX_ALTERNATIVES, logits.shape[1])}, got {top}")
    if not 1e-37 <= temperature <= 1e37:
        raise ValueError(f"token_logprobs: temperature must lie between 1e-37 and 1e37, got {temperature}")
    if logits.is_cuda and _IMPL == "cuda":
        return _k().token_logprobs(logits, tokens, top, temperature)
    return R.token_logprobs(logits, tokens, top, temperature)

# ---------------------------------------------------------------- loss
def cross_entropy(hidden: torch.Tensor, labels: torch.Tensor, weight: torch.Tensor,
                  label_smoothing: float, chunk: int = 2048):
    """Label-smoothed CE of ``hidden @ weight^T`` (tied LM head, ``weight (V,d)``).

    Returns ``(sum_loss, sum_mask)``; the logits are never materialised for the
    whole batch (chunks of ``chunk`` tokens, recomputed in backward)."""
    h = hidden.reshape(-1, hidden.shape[-1])
    lab = labels.reshape(-1)
    if use_cuda(h):
        return _k().cross_entropy(h, lab, weight, label_smoothing)
    import torch.utils.checkpoint as ckpt

    wd = weight.to(h.dtype)

    def piece(hc, lc):
        logits = (hc @ wd.t()).float()
        return R.label_smoothed_ce(logits, lc, label_smoothing)

    tot = h.new_zeros((), dtype=torch.float32)
    cnt = h.new_zeros((), dtype=torch.float32)
    for s in range(0, h.shape[0], chunk):
        if torch.is_grad_enabled():
            a, c = ckpt.checkpoint(piece, h[s:s + chunk], lab[s:s + chunk], use_reentrant=False)
        else:
            a, c = piece(h[s:s + chunk], lab[s:s + chunk])
        tot = tot + a
        cnt = cnt + c
    return tot, cnt
