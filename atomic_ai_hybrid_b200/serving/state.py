"""Per-conversation state of a hybrid model and the mixers' forward over it.

The reference trains only; its layers see whole sequences.  Here every layer keeps, for each of
``slots`` conversations, what its next token needs: the recurrent layers a convolution window of three
rows and a fp32 state of fixed size (``ops.selective_scan``, ``ops.gdn2_recurrent``), MLA its rotated keys
and values (``ops.cached_attention``).  Conversations may start as copies of another one (``fork``): recurrent state is
copied, MLA rows are shared and read once for all of them.  Inside ``serving(...)`` a model's ``forward`` takes ``(1, T)`` packed tokens of several
conversations and its mixers run on this state; everything else in the model is per token already."""
from __future__ import annotations

import contextlib
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
    windows and keys in its compute dtype).  The rest is for models with MLA layers only: ``max_len`` (needed there) bounds the
    rows that a conversation keeps of its own, ``max_positions`` (default ``2 * max_len``) its tokens, those of a conversation
    that it was forked from included.  With ``budget``, a conversation whose rows run out is cut back to that
    many a head (``ops.cache_evict``): its ``recent`` newest tokens (default half of it) and those that got most attention."""

    def __init__(self, model, slots: int, max_len: int = 0, max_positions: int = 0, budget: int = 0, recent: Optional[int] = None):
        if get_tp() is not None or get_cp() is not None:
            raise ValueError("serving runs on one rank's whole model: tensor and context parallelism are for training")
        if any(isinstance(m, MoE) and m.ep_world > 1 for m in model.modules()):
            raise ValueError("serving runs on one rank's whole model: this rank holds a part of the experts only, and every "
                             "layer would wait for the other ranks")
        self.model = model
        p = next(model.parameters())
        self.device, self.dtype, self.slots, self.max_len = p.device, model.compute_dtype, slots, max_len
        # tokens of a conversation, rows of its own that MLA layers keep, the slot that it was forked from (-1: none)
        self.lengths, self.rows, self.prefix = [0] * slots, [0] * slots, [-1] * slots
        self.max_positions, self.budget = max_positions or 2 * max_len, budget
        self.recent = budget // 2 if recent is None else recent
        if budget and not 0 <= self.recent <= budget < max_len:
            raise ValueError(f"budget must be below max_len={max_len} and recent at most budget, got budget={budget}, recent={self.recent}")
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
                if "cos" not in self.__dict__:  # rounded as the training forward's, which multiplies in the compute dtype
                    self.cos, self.sin = (t.to(self.dtype).float() for t in R.rope_cos_sin(self.max_positions, D, device=self.device))
                    # rows and lengths again, where the layers read them
                    self.rows_dev, self.seen_dev = (torch.zeros(slots, dtype=torch.int32, device=self.device) for _ in range(2))
                c = self.layers[m] = dict(k=torch.zeros(slots, H, max_len, D, **kw), v=torch.zeros(slots, H, max_len, D, **kw))
                if budget:
                    c.update(mass=torch.zeros(slots, H, max_len, **f32),
                             held=torch.zeros(slots, H, max_len, dtype=torch.int32, device=self.device))

    @property
    def has_mla(self) -> bool:
        return any("k" in c for c in self.layers.values())

    def on_device(self) -> bool:
        """Whether a token step runs without a host read, as a CUDA graph needs it: every layer's sizes have kernels."""
        from ..ops import kernels as K
        if self.device.type != "cuda" or ops.get_impl() != "cuda":
            return False
        if self.has_mla and self.dtype != torch.bfloat16:
            return False
        return all((not isinstance(m, Mamba2) or m.cfg.d_state in K.SCAN_STATES)
                   and (not isinstance(m, GatedDeltaNet2) or m.d_head in K.RECURRENT_HEADS)
                   and (not isinstance(m, MLA) or m.cfg.d_model // m.cfg.n_heads in K.ATTENTION_HEADS)
                   and (not isinstance(m, MoE) or m.has_kernels(self.dtype)) for m in self.model.modules())

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for c in self.layers.values() for t in c.values())

    def check_slots(self, slots: List[int]) -> None:
        if len(set(slots)) != len(slots) or any(not 0 <= s < self.slots for s in slots):
            raise ValueError(f"slots must be different and below {self.slots}: {slots}")

    def reset(self, slots: List[int]) -> None:
        """Makes the conversations in ``slots`` new ones."""
        self.check_slots(slots)
        self._check_unshared(slots, besides=slots)
        idx = torch.tensor(slots, dtype=torch.long, device=self.device)
        for cache in self.layers.values():
            for name in ("conv", "state"):
                if name in cache:
                    cache[name][idx] = 0
        for s in slots:
            self.lengths[s], self.rows[s], self.prefix[s] = 0, 0, -1
        self._rows_to_device(slots)

    def _rows_to_device(self, slots: List[int]) -> None:
        if self.has_mla and slots:
            now = torch.tensor([[s, self.rows[s], self.lengths[s]] for s in slots], dtype=torch.int32).to(self.device)
            idx = now[:, 0].long()
            self.rows_dev[idx], self.seen_dev[idx] = now[:, 1], now[:, 2]

    def _check_unshared(self, slots: List[int], besides: List[int] = ()) -> None:
        """A conversation whose rows others read stays as it is while they do."""
        mine, free = set(slots), set(besides)
        by = {p: s for s, p in enumerate(self.prefix) if p in mine and s not in free}
        if by:
            raise ValueError(f"slot {min(by)} is shared: the conversation in slot {by[min(by)]} was forked from it and reads its rows")

    def fork(self, source: int, slots: List[int]) -> None:
        """Makes the conversations in ``slots`` new ones that go on from the one in ``source``.  Recurrent layers' state is
        copied; MLA layers' rows are not: as long as these conversations live, ``source`` adds no tokens, and it must not have been
        forked from another one itself."""
        self.check_slots(slots)
        self.check_slots([source])
        if source in slots:
            raise ValueError(f"slot {source} cannot be forked into itself")
        if self.has_mla and self.prefix[source] >= 0:
            raise ValueError(f"the conversation in slot {source} was forked from slot {self.prefix[source]}: its rows are not all its own")
        self.reset(slots)
        idx = torch.tensor(slots, dtype=torch.long, device=self.device)
        for cache in self.layers.values():
            for name in ("conv", "state"):
                if name in cache:
                    cache[name][idx] = cache[name][source].clone()
        for s in slots:
            self.lengths[s] = self.lengths[source]
            self.prefix[s] = source if self.has_mla else -1
        self._rows_to_device(slots)

    def check_room(self, slots: List[int], lens: List[int], fresh: bool = False, before: int = 0) -> List[int]:
        """Raises where MLA layers cannot hold ``lens`` more tokens (``fresh``: of new conversations, behind ``before`` shared ones);
        returns the slots that are to be cut back for them."""
        if not self.has_mla:
            return []
        if not fresh:
            self._check_unshared(slots)
        cut = []
        for s, n in zip(slots, lens):
            if (before if fresh else self.lengths[s]) + n > self.max_positions:
                raise ValueError(f"a conversation would grow past max_positions={self.max_positions}")
            if (0 if fresh else self.rows[s]) + n > self.max_len:
                if not self.budget or fresh or min(self.rows[s], self.budget) + n > self.max_len:
                    raise ValueError(f"a conversation would grow past max_len={self.max_len}")
                cut.append(s)
        return cut

    def cut_back(self, slots: List[int]) -> None:
        """Cuts the MLA rows of the conversations in ``slots`` back to ``budget`` a head."""
        if not slots:
            return
        self.check_slots(slots)
        self._check_unshared(slots)
        if not self.budget:
            raise ValueError("cutting back needs a budget")
        which = torch.tensor(slots, dtype=torch.int32, device=self.device)
        for c in self.layers.values():
            if "mass" in c:
                ops.cache_evict(c["k"], c["v"], c["mass"], c["held"], self.rows_dev, self.seen_dev, self.budget, recent=self.recent,
                                slots=which)
        for s in slots:
            self.rows[s] = min(self.rows[s], self.budget)
        self._rows_to_device(slots)


class _Call:
    """One forward over packed tokens: sequence ``i`` adds ``lens[i]`` tokens to slot ``slots[i]``."""

    def __init__(self, state: DecodeState, slots: List[int], lens: Optional[List[int]], slots_dev=None, prefix_dev=None):
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
        self.prefix_dev = prefix_dev
        if prefix_dev is None and any(state.prefix[s] >= 0 for s in slots):
            self.prefix_dev = torch.tensor([state.prefix[s] for s in slots], dtype=torch.int32).to(dev)
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
        self._check_rows(x)
        st, c = self.state, self.state.layers[mod]
        q, lat = mod.W_q(x)[0], mod.W_kv_down(x)
        o = ops.cached_attention(q, mod.W_k_up(lat)[0], mod.W_v_up(lat)[0], c["k"], c["v"], st.rows_dev, cos=st.cos, sin=st.sin,
                                 cu_seqlens=self.cu, slots=self.slots_dev, prefix=self.prefix_dev, seen=st.seen_dev,
                                 mass=c.get("mass"), held=c.get("held"))
        return mod.W_o(mod.attn_out_norm(o[None]))

    def advance(self) -> None:
        """Moves the conversations past this call's tokens."""
        st = self.state
        for s, n in zip(self.slots, self.lens or [1] * len(self.slots)):
            st.lengths[s] += n
            st.rows[s] += n
        if st.has_mla:
            n = torch.ones_like(self.slots_dev) if self.cu is None else self.cu[1:] - self.cu[:-1]
            st.rows_dev.index_add_(0, self.slots_dev, n)
            st.seen_dev.index_add_(0, self.slots_dev, n)


@contextlib.contextmanager
def serving(state: DecodeState, slots: List[int], lens: Optional[List[int]] = None, slots_dev=None, fresh: bool = False,
            prefix_dev=None):
    """Runs a model's forwards on ``state``: ``(1, T)`` tokens of ``len(slots)`` conversations packed one
    after another, ``lens[i]`` of them each (None: one each; ``fresh``: as new conversations).  ``slots_dev`` is
    ``slots`` as an int32 tensor on the device, where the caller has it, ``prefix_dev`` the slots that they were forked from.  It holds for the thread that enters it; a
    state serves one call at a time."""
    if get_serving() is not None:
        raise RuntimeError("serving(...) is not nested")
    state.check_slots(slots)
    if lens is not None and (len(lens) != len(slots) or min(lens, default=1) < 1):
        raise ValueError("every sequence of a call adds at least one token")
    cut = state.check_room(slots, lens or [1] * len(slots), fresh)
    if fresh:
        state.reset(slots)
    state.cut_back(cut)
    call = _Call(state, slots, lens, slots_dev, prefix_dev)
    token = serving_call.enter(call)
    try:
        yield call
        call.advance()
    finally:
        serving_call.leave(token)
