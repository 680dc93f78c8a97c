"""Training loss (reference ``compute_loss``, `optimizer.py:315-430`).

``total = ce + aux_coef * sum(aux) + z_coef * sum(z) + collinearity_coef * sum(collinearity)``
where the router terms are summed over the MoE layers and ``ce`` is the
label-smoothed cross entropy of the tied LM head (mask label ``-100``).  In
evaluation (``deterministic=True``) the router terms are zero, as in the
reference.  Returns ``(total, aux_info)`` with the reference's 14 aux keys.
"""
from __future__ import annotations

from typing import Dict, List, Optional

import torch

from .. import ops

ROUTER_COLLINEARITY_COEF = 0.08


def _stack(stats: List[Dict], key: str) -> Optional[torch.Tensor]:
    vals = [s[key] for s in stats if key in s]
    return torch.stack([v.float() for v in vals]) if vals else None


def compute_loss(model, batch: Dict[str, torch.Tensor], deterministic: bool = False,
                 ce_chunk_size: int = 2048, collinearity_coef: Optional[float] = None):
    cfg = model.cfg
    hidden, stats = model(batch["input_ids"], return_hidden=True)
    labels = model.token_shard(batch["labels"]) if hasattr(model, "token_shard") else batch["labels"]
    sum_loss, sum_mask = ops.cross_entropy(hidden, labels, model.lm_weight(),
                                           cfg.label_smoothing, ce_chunk_size)
    ce = sum_loss / sum_mask.clamp_min(1.0)
    ce = torch.nan_to_num(ce, nan=0.0, posinf=1e4, neginf=0.0)
    zero = ce.new_zeros(())
    if deterministic or not stats:
        aux = z = coll = zero
    else:
        aux = _stack(stats, "aux_loss").sum()
        z = _stack(stats, "z_loss").sum()
        coll = _stack(stats, "router_collinearity").sum()
    coef = ROUTER_COLLINEARITY_COEF if collinearity_coef is None else collinearity_coef
    total = ce + cfg.router_aux_loss_coef * aux + cfg.router_z_loss_coef * z + coef * coll
    mc = _stack(stats, "router_max_cos")
    info = {
        "ce_loss": ce.detach(),
        "aux_loss": aux.detach(),
        "z_loss": z.detach(),
        "expert_utilization": _stack(stats, "expert_utilization"),
        "moe_dropped_ratio": _stack(stats, "moe_dropped_ratio"),
        "router_temp": _stack(stats, "router_temp"),
        "min_col_norm": _stack(stats, "min_col_norm"),
        "max_abs_logit_preclip": _stack(stats, "max_abs_logit_preclip"),
        "norm_x_mean": _stack(stats, "norm_x_mean"),
        "norm_x_max": _stack(stats, "norm_x_max"),
        "norm_x_min": _stack(stats, "norm_x_min"),
        "router_max_cos_per_layer": mc,
        "router_max_cos": mc.max() if mc is not None else zero,
        "assignment_frac": _stack(stats, "assignment_frac"),
    }
    return total, info


class _HeadScores(torch.autograd.Function):
    """``ops.token_logprobs`` of ``h @ weight^T``, whose logits exist for ``chunk`` rows at a time, in the backward again.  The
    weight's gradient is summed over all rows in fp32, in the parameter's accumulator where it has one, and else rounded once."""

    @staticmethod
    def forward(ctx, h, labels, weight, temperature, chunk):
        ctx.save_for_backward(h, labels)
        ctx.weight, ctx.temperature, ctx.chunk = weight, temperature, chunk
        w = weight.to(h.dtype)
        parts = [ops.token_logprobs(h[s:s + chunk] @ w.t(), labels[s:s + chunk], temperature=temperature)
                 for s in range(0, max(1, h.shape[0]), chunk)]
        return tuple(torch.cat(t) for t in zip(*parts))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, ge):
        h, labels = ctx.saved_tensors
        weight, chunk = ctx.weight, ctx.chunk
        w = weight.detach().to(h.dtype)
        dh = torch.empty_like(h) if ctx.needs_input_grad[0] else None
        direct = sums = None
        if ctx.needs_input_grad[2]:
            direct = getattr(weight, "_ahb_grad_acc", None)
            own = direct is None or direct.dtype != torch.float32
            sums = torch.zeros(weight.shape, dtype=torch.promote_types(h.dtype, torch.float32), device=h.device) if own else direct.view(weight.shape)
        for s in range(0, h.shape[0], chunk):
            hc = h[s:s + chunk]
            with torch.enable_grad():
                logits = (hc @ w.t()).detach().requires_grad_()
                out = ops.token_logprobs(logits, labels[s:s + chunk], temperature=ctx.temperature)
            d, = torch.autograd.grad(out, [logits], [g[s:s + chunk], ge[s:s + chunk]])
            if dh is not None:
                torch.mm(d, w, out=dh[s:s + chunk])
            if sums is None:
                continue
            if ops.use_cuda(h) and h.dtype == torch.bfloat16 and sums.dtype == torch.float32:
                from ..ops import kernels as K
                K._wgrad_acc(sums, d, hc)
            else:
                sums.addmm_(d.t().to(sums.dtype), hc.to(sums.dtype))
        dw = None
        if sums is not None and direct is None:
            dw = sums.to(weight.dtype)
        elif sums is not None and direct.dtype != torch.float32:
            direct.view(weight.shape).add_(sums)
        return dh, None, dw, None, None


def token_scores(model, batch: Dict[str, torch.Tensor], temperature: float = 1.0, chunk: int = 2048):
    """``(logprobs, entropy)``, fp32 and shaped like ``batch["labels"]`` (under tensor or context parallelism like the rank's shard of them):
    the log-probability of every label under the model and the entropy of the distribution that it is drawn from, with
    gradients (``ops.token_logprobs``), for objectives on the answers themselves (preference pairs, policy gradients).  Labels of -100
    have log-probability 0 and no gradient.  As in ``compute_loss`` the logits are made ``chunk`` tokens at a time and again in
    the backward, and the head's gradient is summed in fp32; logits are rounded to the hidden states' type, and so are their gradients."""
    hidden, _ = model(batch["input_ids"], return_hidden=True)
    labels = model.token_shard(batch["labels"]) if hasattr(model, "token_shard") else batch["labels"]
    lp, entropy = _HeadScores.apply(hidden.reshape(-1, hidden.shape[-1]), labels.reshape(-1), model.lm_weight(), temperature, chunk)
    return lp.view(labels.shape), entropy.view(labels.shape)
