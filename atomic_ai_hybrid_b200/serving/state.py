"""Per-conversation state of a hybrid model and the mixers' forward over it.

The reference trains only; its layers see whole sequences.  Here every layer keeps, for each of
``slots`` conversations, what its next token needs: the recurrent layers a convolution window of three
rows and a fp32 state of fixed size (``ops.selective_scan``, ``ops.gdn2_recurrent``), MLA its rotated keys
and values.  Inside ``serving(...)`` a model's ``forward`` takes ``(1, T)`` packed tokens of several
conversations and its mixers run on this state; everything else in the model is per token already."""
from __future__ import annotations

import contextlib
import math
from typing import Dict, List, Optional

import torch
import torch.nn.functional as F

from .. import ops
from ..models.mixers import MLA, GatedDeltaNet2, Mamba2
from ..models.moe import MoE
from ..ops import reference as R
from ..parallel.cp import get_cp
from ..parallel.tp import get_tp
from ..utils import serving_call
from ..utils.serving_call import get_serving

# GDN-2 prompts of at least this many tokens, in at most this many (sequence, head) pairs, run on the chunked
# training scan.  It runs a head's chunks side by side, but each call pays 0.9 ms of separate launches for padding,
# convolutions and gates; token by token a head takes 1.3 us a token on an SM of its own.  Whole mixer of
# 16 heads of 128, chunked against token by token: 1 sequence of 512 tokens 1.20 and 0.94 ms, 768 1.21 and 1.27,
# 4096 1.8 and 5.7; 4 sequences of 768 1.50 and 1.40, 1024 1.65 and 1.75, 4096 4.4 and 6.3; 6 of 1024 2.06 and 1.84,
# 4096 6.4 and 6.8; 32 of 1024 8.3 and 5.5.
# The chunked scan multiplies bf16 operands, as in the training forward that the weights come from: its state after 800
# tokens is 4e-3 off the 64-bit one, token by token (fp32 throughout) 1e-7.  So which form a prompt took, by its length
# and by how many others came with it, shows in its answer's last digits; the later tokens add nothing to it.
GDN_CHUNKED_FROM, GDN_CHUNKED_HEADS = 768, 64


class DecodeState:
    """State of ``slots`` conversations for every mixer of ``model`` (on its device, convolution
    windows and keys in its compute dtype).  ``max_len`` bounds a conversation's tokens and is needed for
    models with MLA layers only."""

    def __init__(self, model, slots: int, max_len: int = 0):
        if get_tp() is not None or get_cp() is not None:
            raise ValueError("serving runs on one rank's whole model: tensor and context parallelism are for training")
        if any(isinstance(m, MoE) and m.ep_world > 1 for m in model.modules()):
            raise ValueError("serving runs on one rank's whole model: this rank holds a part of the experts only, and every "
                             "layer would wait for the other ranks")
        self.model = model
        p = next(model.parameters())
        self.device, self.dtype, self.slots, self.max_len = p.device, model.compute_dtype, slots, max_len
        self.lengths = [0] * slots
        self.layers: Dict[torch.nn.Module, dict] = {}
        kw = dict(device=self.device, dtype=self.dtype)
        f32 = dict(device=self.device, dtype=torch.float32)
        for m in model.modules():
            if isinstance(m, Mamba2):
                H, C = m.n_heads, m.cfg.d_inner
                self.layers[m] = dict(conv=torch.zeros(slots, 3, C, **kw),
                                      state=torch.zeros(slots, H, C // H, m.cfg.d_state, **f32))
            elif isinstance(m, GatedDeltaNet2):
                H, D = m.n_heads, m.d_head
                self.layers[m] = dict(conv=torch.zeros(slots, 3, 3, H * D, **kw), state=torch.zeros(slots, H, D, D, **f32))
            elif isinstance(m, MLA):
                if max_len <= 0:
                    raise ValueError("a model with MLA layers keeps keys and values: max_len must be given")
                H, D = m.n_heads, m.cfg.d_model // m.cfg.n_heads
                if "cos" not in self.__dict__:
                    self.cos, self.sin = R.rope_cos_sin(max_len, D, device=self.device)
                self.layers[m] = dict(k=torch.zeros(slots, max_len, H, D, **kw), v=torch.zeros(slots, max_len, H, D, **kw))

    @property
    def has_mla(self) -> bool:
        return any("k" in c for c in self.layers.values())

    def on_device(self) -> bool:
        """Whether a token step runs without a host read, as a CUDA graph needs it: every layer's sizes have kernels."""
        from ..ops import kernels as K
        if self.device.type != "cuda" or ops.get_impl() != "cuda" or self.has_mla:
            return False
        return all((not isinstance(m, Mamba2) or m.cfg.d_state in K.SCAN_STATES)
                   and (not isinstance(m, GatedDeltaNet2) or m.d_head in K.RECURRENT_HEADS)
                   and (not isinstance(m, MoE) or m.has_kernels(self.dtype)) for m in self.model.modules())

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for c in self.layers.values() for t in c.values())

    def check_slots(self, slots: List[int]) -> None:
        if len(set(slots)) != len(slots) or any(not 0 <= s < self.slots for s in slots):
            raise ValueError(f"slots must be different and below {self.slots}: {slots}")

    def reset(self, slots: List[int]) -> None:
        """Makes the conversations in ``slots`` new ones."""
        self.check_slots(slots)
        idx = torch.tensor(slots, device=self.device)
        for cache in self.layers.values():
            for name in ("conv", "state"):
                if name in cache:
                    cache[name][idx] = 0
        for s in slots:
            self.lengths[s] = 0


class _Call:
    """One forward over packed tokens: sequence ``i`` adds ``lens[i]`` tokens to slot ``slots[i]``."""

    def __init__(self, state: DecodeState, slots: List[int], lens: Optional[List[int]], slots_dev=None):
        self.state, self.slots, self.lens = state, slots, lens
        dev = state.device
        self.slots_dev = slots_dev if slots_dev is not None else torch.tensor(slots, dtype=torch.int32, device=dev)
        self.cu = None
        if lens is not None:
            ends = [0]
            for n in lens:
                ends.append(ends[-1] + n)
            self.starts = ends
            self.cu = torch.tensor(ends, dtype=torch.int32, device=dev)
        self._pad = self._rates = None

    def _check_rows(self, x: torch.Tensor) -> None:
        want = len(self.slots) if self.lens is None else sum(self.lens)
        if x.shape[0] != 1 or x.shape[1] != want:
            raise ValueError(f"this call has {want} tokens packed in one row, the forward {x.shape[1]} in {x.shape[0]}")

    # ------------------------------------------------------------ Mamba2
    def _decay_rates(self):
        """``A = -exp(A_log)`` of every Mamba2 layer, from the weights as they are now: four launches a call for all."""
        if self._rates is None:
            mods = [m for m in self.state.layers if isinstance(m, Mamba2)]
            logs = torch._foreach_clamp_min([m.A_log.detach().float() for m in mods], -20.0)
            self._rates = dict(zip(mods, torch._foreach_neg(torch._foreach_exp(torch._foreach_clamp_max(logs, 20.0)))))
        return self._rates

    def mamba2(self, mod: Mamba2, x: torch.Tensor) -> torch.Tensor:
        self._check_rows(x)
        c = self.state.layers[mod]
        xz = mod.in_projection(x)
        di = xz.shape[-1] // 2
        x_bc, res = xz[..., :di], xz[..., di:]
        if ops.use_cuda(x) and x.dtype == torch.bfloat16:
            from ..ops import kernels as K
            Bm, Cm, dt = K.linear_multi(x_bc, [(m.kernel, m.bias) for m in (mod.B_proj, mod.C_proj, mod.dt_proj)])
        else:
            Bm, Cm, dt = mod.B_proj(x_bc), mod.C_proj(x_bc), mod.dt_proj(x_bc)
        y = ops.selective_scan(x_bc[0], dt[0], self._decay_rates()[mod], Bm[0], Cm[0], mod.conv_w.detach(), mod.conv_b.detach(), c["conv"],
                               c["state"], cu_seqlens=self.cu, slots=self.slots_dev)[None]
        if ops.use_cuda(x) and x.dtype == torch.bfloat16:
            from ..ops import kernels as K
            if K.row_fusable(di):
                return mod.out_projection(K.norm_gate(y, res, mod.ssm_out_norm.scale, 1e-6, oclip=3e2))
        return mod.out_projection((mod.ssm_out_norm(y) * F.silu(res)).clamp(-3e2, 3e2))

    # ------------------------------------------------------------ GDN-2
    def gdn2(self, mod: GatedDeltaNet2, x: torch.Tensor) -> torch.Tensor:
        self._check_rows(x)
        c = self.state.layers[mod]
        *ins, og = mod.projections(x)
        if (self.lens is not None and max(self.lens) >= GDN_CHUNKED_FROM and len(self.lens) * mod.n_heads <= GDN_CHUNKED_HEADS
                and mod.d_head == 128 and ops.use_cuda(x)):
            o = self._gdn2_chunked(mod, c, ins)
        else:
            convs = [mod.q_conv_w, mod.k_conv_w, mod.v_conv_w], [mod.q_conv_b, mod.k_conv_b, mod.v_conv_b]
            o = ops.gdn2_recurrent(*(t[0] for t in ins), [w.detach() for w in convs[0]], [b.detach() for b in convs[1]],
                                   mod.decay_a.detach(), c["conv"], c["state"], cu_seqlens=self.cu, slots=self.slots_dev)
        o = o[None]
        if ops.use_cuda(x) and x.dtype == torch.bfloat16:
            from ..ops import kernels as K
            if K.row_fusable(o.shape[-1]):
                return mod.out_projection(K.norm_gate(o, og, mod.out_norm.scale, 1e-6, zclip=1e2))
        return mod.out_projection(mod.out_norm(o) * F.silu(og.clamp(-1e2, 1e2)))

    def _padded(self):
        """Packed rows as ``(sequences, tokens up to a multiple of 64)``, and where a token is."""
        if self._pad is None:
            L = -(-max(self.lens) // 64) * 64
            n = torch.tensor(self.lens, device=self.state.device)
            at = torch.arange(L, device=self.state.device)
            has = at < n[:, None]
            self._pad = torch.where(has, self.cu[:-1, None].long() + at, 0), has, n
        return self._pad

    def _gdn2_chunked(self, mod, c, ins):
        """Long prompts of few heads: the training kernels' convolution and chunked scan on padded rows, from and into the state."""
        row, has, n = self._padded()
        H, D = mod.n_heads, mod.d_head
        B, L = row.shape
        slots = self.slots_dev.long()
        shp = (B, L, H, D)
        qkv = []
        for m, (name, clip) in enumerate((("q", None), ("k", None), ("v", 50.0))):
            ext = torch.cat([c["conv"][slots, m], ins[m][0][row] * has[..., None]], 1)  # the window leads, as earlier tokens
            w, b = getattr(mod, f"{name}_conv_w"), getattr(mod, f"{name}_conv_b")
            qkv.append(ops.conv1d(ext, w, b, silu=True, clip=clip)[:, 3:].reshape(shp))
            last = (n[:, None] + torch.arange(3, device=n.device))[..., None].expand(-1, -1, ext.shape[2])
            c["conv"][slots, m] = ext.gather(1, last)
        live = has[..., None, None]
        q, k = (R.safe_l2norm(t, 1e-12) for t in qkv[:2])
        b, w, f = (t[0][row].view(shp) for t in ins[3:])
        g = -torch.exp(mod.decay_a.float().clamp(-20.0, 20.0))[:, None] * F.softplus(f.float())
        g = torch.nan_to_num(g, nan=0.0, posinf=0.0, neginf=-20.0).clamp(-1e3, 1e3)
        # a row past a sequence's end neither decays, erases nor writes
        o, hf = ops.gdn2(q, k * live, qkv[2], torch.sigmoid(w) * live, torch.sigmoid(b), g * live, 1.0, mod.cfg.gdn_chunk,
                         h0=c["state"][slots], return_final=True)
        c["state"][slots] = hf
        return o.reshape(B, L, H * D)[has].to(ins[0].dtype)

    # ------------------------------------------------------------ MLA
    def mla(self, mod: MLA, x: torch.Tensor) -> torch.Tensor:
        """Keys and values kept rotated per slot; the products are PyTorch's attention, as under
        context parallelism."""
        self._check_rows(x)
        st, c = self.state, self.state.layers[mod]
        H, D = mod.n_heads, mod.cfg.d_model // mod.cfg.n_heads
        lens = self.lens or [1] * len(self.slots)
        pos = torch.cat([torch.arange(st.lengths[s], st.lengths[s] + n) for s, n in zip(self.slots, lens)]).to(x.device)
        which = torch.repeat_interleave(torch.tensor(self.slots), torch.tensor(lens)).to(x.device)
        cos, sin = st.cos[pos][:, None], st.sin[pos][:, None]
        q, lat = mod.W_q(x)[0], mod.W_kv_down(x)
        q = R.apply_rope(q.view(-1, H, D), cos, sin)
        k = R.apply_rope(mod.W_k_up(lat)[0].view(-1, H, D), cos, sin)
        v = mod.W_v_up(lat)[0].view(-1, H, D)
        q, k, v = (R.sanitize(t, 1e3) for t in (q, k, v))
        c["k"][which, pos], c["v"][which, pos] = k, v
        out, at = [], 0
        for s, n in zip(self.slots, lens):
            end = st.lengths[s] + n
            keep = torch.arange(end, device=x.device)[None] <= pos[at:at + n, None]
            out.append(F.scaled_dot_product_attention(q[at:at + n].transpose(0, 1)[None], c["k"][s, :end].transpose(0, 1)[None],
                                                      c["v"][s, :end].transpose(0, 1)[None], attn_mask=keep,
                                                      scale=1.0 / math.sqrt(D))[0].transpose(0, 1))
            at += n
        o = torch.cat(out).reshape(1, -1, H * D)
        return mod.W_o(mod.attn_out_norm(o))


@contextlib.contextmanager
def serving(state: DecodeState, slots: List[int], lens: Optional[List[int]] = None, slots_dev=None, fresh: bool = False):
    """Runs a model's forwards on ``state``: ``(1, T)`` tokens of ``len(slots)`` conversations packed one
    after another, ``lens[i]`` of them each (None: one each; ``fresh``: as new conversations).  ``slots_dev`` is
    ``slots`` as an int32 tensor on the device, where the caller has it.  It holds for the thread that enters it; a
    state serves one call at a time."""
    if get_serving() is not None:
        raise RuntimeError("serving(...) is not nested")
    state.check_slots(slots)
    if lens is not None and (len(lens) != len(slots) or min(lens, default=1) < 1):
        raise ValueError("every sequence of a call adds at least one token")
    if state.has_mla and any((0 if fresh else state.lengths[s]) + n > state.max_len
                             for s, n in zip(slots, lens or [1] * len(slots))):
        raise ValueError(f"a conversation would grow past max_len={state.max_len}")
    if fresh:
        state.reset(slots)
    call = _Call(state, slots, lens, slots_dev)
    token = serving_call.enter(call)
    try:
        yield call
        for s, n in zip(slots, lens or [1] * len(slots)):
            state.lengths[s] += n
    finally:
        serving_call.leave(token)
