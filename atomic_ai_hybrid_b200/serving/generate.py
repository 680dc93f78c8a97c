"""Token generation from a hybrid model: prompts, then one token at a time, each drawn by ``ops.sample``."""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from .. import ops
from ..models.hybrid import flax_path
from ..optim.store import default_keep_fp32
from .state import DecodeState, serving


def load_weights(model, root: str, slot: str = "latest", step: Optional[int] = None) -> List[str]:
    """Fills ``model`` from a training checkpoint (any parallel layout's files; the parameters keep their
    dtypes); returns the names that the checkpoint does not hold.  One that holds a tensor of another shape is of
    another model: that is an error, and nothing is loaded."""
    from ..ckpt.manager import CheckpointManager, _assemble_tp, _lookup

    mgr = CheckpointManager(root, slot)
    step = mgr.latest_step() if step is None else step
    if step is None:
        raise FileNotFoundError(f"no checkpoint in {root}/{slot}")
    params, _, _ = mgr.load_tensors(step)
    found, absent, other = [], [], []
    for n, p in model.named_parameters():
        t = _lookup(params, flax_path(n), None)
        if t is None:
            t = _assemble_tp(params, flax_path(n))
        if t is None:
            absent.append(n)
        elif tuple(t.shape) != tuple(p.shape):
            other.append(f"{n} {tuple(t.shape)} for {tuple(p.shape)}")
        else:
            found.append((p, t))
    if other:
        raise ValueError(f"the checkpoint in {root}/{slot} has {len(other)} parameters of another shape: {', '.join(other[:8])}")
    with torch.no_grad():
        for p, t in found:
            p.copy_(t)
    return absent


def compute_weights(model):
    """Keeps ``model``'s matrices in its compute dtype from here on, those that training computes with in fp32 (router,
    norms, biases) apart: half the memory, and no rounding at every token.  Parameters that a trainer's store holds
    already are its views, and stay.  Returns ``model``."""
    for n, p in model.named_parameters():
        if not default_keep_fp32(n, p) and not hasattr(p, "_ahb_grad_acc"):
            p.data = p.data.to(model.compute_dtype)
    return model


SCORE_LOGITS = 1 << 28  # logits that ``Generator.score`` makes at a time (half a GB in bf16)
MAX_GRAPHS = 8  # captured token steps that a Generator keeps, one per batch size; a capture launches the step twice


class Generator:
    """Answers up to ``max_sequences`` prompts at a time.

    ``model`` stays as it is, in training mode or not and owned by a trainer or not: its weights are read where they
    are at every token, matrices of another dtype than the compute dtype are rounded on the way (``compute_weights``
    keeps them rounded).  ``max_len`` bounds prompt plus answer for models with MLA layers, a common prefix apart; with
    ``kv_budget`` longer conversations go on up to ``max_positions`` tokens, with that many rows a head once the rows run out:
    the ``kv_recent`` newest and those that got most attention (``DecodeState``).  On a GPU, models whose sizes all have
    kernels replay the token step from one CUDA graph per batch size; others launch it."""

    def __init__(self, model, max_sequences: int, max_len: int = 0, cuda_graph: bool = True, max_positions: int = 0,
                 kv_budget: int = 0, kv_recent: Optional[int] = None):
        self.model = model
        p = next(model.parameters())
        self.device = p.device
        self.state = DecodeState(model, max_sequences, max_len, max_positions, kv_budget, kv_recent)
        self.cuda_graph = cuda_graph
        self._graphs, self._captured, self._rows = {}, None, None

    # ------------------------------------------------------------ forwards
    def _logits(self, h: torch.Tensor) -> torch.Tensor:
        return h @ self.model.lm_weight().to(h.dtype).t()

    @torch.no_grad()
    def prefill(self, prompts: Sequence[Sequence[int]], slots: List[int], fresh: bool = True) -> torch.Tensor:
        """Reads ``prompts`` into ``slots`` (``fresh``: as new conversations) and returns the logits
        ``(prompts, vocabulary)`` after their last tokens."""
        h, last = self._read(prompts, slots, fresh)
        return self._logits(h[last])

    def _read(self, prompts: Sequence[Sequence[int]], slots: List[int], fresh: bool):
        """The hidden rows of ``prompts``, packed, and where each one's last row is."""
        lens = [len(p) for p in prompts]
        ids = self._ids(prompts).to(self.device)
        with serving(self.state, slots, lens, fresh=fresh) as call:
            h, _ = self.model(ids[None])
            last = call.cu[1:].long() - 1
        return h[0], last

    def _ids(self, prompts: Sequence[Sequence[int]]) -> torch.Tensor:
        ids = torch.cat([torch.as_tensor(p, dtype=torch.long) for p in prompts])
        if ids.numel() and not 0 <= int(ids.min()) <= int(ids.max()) < self.model.cfg.vocab_size:
            raise ValueError(f"prompts need token ids of the vocabulary, [0, {self.model.cfg.vocab_size})")
        return ids

    def fork(self, source: int, slots: List[int]) -> None:
        """Makes the conversations in ``slots`` new ones that go on from the one in ``source`` (``DecodeState.fork``)."""
        self.state.fork(source, slots)

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, slots: List[int]) -> torch.Tensor:
        """One token for each conversation in ``slots``; returns the logits ``(slots, vocabulary)``."""
        with serving(self.state, slots):
            h, _ = self.model(tokens.to(self.device)[None])
        return self._logits(h[0])

    def _graph_step(self, slots: List[int]):
        """The token step over ``slots`` and its sampling as one graph; returns it with its buffers."""
        where = [(p.data_ptr(), p.dtype) for p in self.model.parameters()]
        if where != self._captured:  # a graph reads the weights by address: they have moved since
            self._graphs.clear()
            self._captured = where
        key = tuple(slots), tuple(self.state.prefix[s] for s in slots)
        if key not in self._graphs:
            while len(self._graphs) >= MAX_GRAPHS:  # the one that was used least recently
                self._graphs.pop(next(iter(self._graphs)))
            B, V, dev = len(slots), self.model.cfg.vocab_size, self.device
            if self._rows is None:  # what the graphs read by address: rows of the same buffers, as they run one at a time
                n = self.state.slots
                self._rows = dict(tokens=torch.zeros(n, dtype=torch.long, device=dev), noise=torch.ones(n, V, device=dev),
                                  temperature=torch.ones(n, device=dev), top_k=torch.zeros(n, dtype=torch.int32, device=dev),
                                  top_p=torch.ones(n, device=dev), min_p=torch.zeros(n, device=dev))
                # one stream, of the model's device, for every capture: the allocator keeps a stream's memory for it
                self._pool, self._side = torch.cuda.graph_pool_handle(), torch.cuda.Stream(device=dev)
            buf = {name: t[:B] for name, t in self._rows.items()}
            buf["slots"], buf["prefix"] = (torch.tensor(s, dtype=torch.int32, device=dev) for s in key)
            if max(key[1]) < 0:
                buf["prefix"] = None

            def run():
                with serving(self.state, slots, slots_dev=buf["slots"], prefix_dev=buf["prefix"]):
                    h, _ = self.model(buf["tokens"][None])
                t, lp = ops.sample(self._logits(h[0]), buf["noise"], buf["temperature"], buf["top_k"], buf["top_p"], buf["min_p"])
                buf["tokens"].copy_(t.clamp(min=0))
                return t, lp

            # Warm up and capture on a copy of what the step changes.  Both runs count as a conversation's first token on the host, so that
            # neither asks for room or cuts anything back; where the device's own counts leave no room, the warm-up's tokens are padding.
            st = self.state
            st.check_room(slots, [1] * B)
            changed = [c[n] for c in st.layers.values() for n in ("conv", "state", "mass", "held") if n in c]
            changed += [st.rows_dev, st.seen_dev] if st.has_mla else []
            kept = [t.clone() for t in changed]
            lengths, rows = list(st.lengths), list(st.rows)
            side = self._side
            side.wait_stream(torch.cuda.current_stream(dev))
            graph = torch.cuda.CUDAGraph()
            try:
                st.lengths, st.rows = [0] * st.slots, [0] * st.slots
                with torch.cuda.stream(side):
                    run()
                torch.cuda.current_stream(dev).wait_stream(side)
                st.lengths, st.rows = [0] * st.slots, [0] * st.slots
                with torch.cuda.graph(graph, pool=self._pool, stream=side):
                    buf["out"] = run()
            finally:
                torch.cuda.current_stream(dev).wait_stream(side)
                for t, k in zip(changed, kept):
                    t.copy_(k)
                st.lengths, st.rows = lengths, rows
        else:
            graph, buf = self._graphs.pop(key)
        self._graphs[key] = graph, buf
        return graph, buf

    def _check_waits(self) -> None:
        """Where the host has waited for the device anyway: no answers from kernels that gave up (``prefill`` and ``step`` do not wait)."""
        if self.device.type == "cuda" and ops.get_impl() == "cuda":
            from ..ops import kernels as K
            K.check_waits()

    # ------------------------------------------------------------ scores
    def _check_prompts(self, prompts, prefix) -> None:
        room = self.state.slots - (prefix is not None)
        if not 1 <= len(prompts) <= room:
            raise ValueError(f"{len(prompts)} prompts, room for {room}")
        if any(len(p) == 0 for p in prompts) or prefix is not None and len(prefix) == 0:
            raise ValueError("a prompt needs at least one token")

    def _check_new(self, prompts, prefix) -> None:
        """What reading ``prompts`` and ``prefix`` would be refused for, before any conversation is changed."""
        before = 0 if prefix is None else len(prefix)
        self._ids(prompts if prefix is None else [prefix, *prompts])
        if before:
            self.state.check_room([len(prompts)], [before], fresh=True)
        self.state.check_room(list(range(len(prompts))), [len(p) for p in prompts], fresh=True, before=before)

    def _read_prefix(self, prefix: Sequence[int], B: int) -> torch.Tensor:
        """Reads ``prefix`` into slot ``B`` and forks slots 0 to ``B - 1`` from it; returns its last hidden row."""
        self.state.reset(list(range(B + 1)))
        h, last = self._read([prefix], [B], True)
        self.state.fork(B, list(range(B)))
        return h[last]

    @torch.no_grad()
    def score(self, sequences: Sequence[Sequence[int]], top: int = 0, temperature: float = 1.0,
              prefix: Optional[Sequence[int]] = None):
        """How likely the model finds ``sequences`` (lists of token ids, at most ``max_sequences`` non-empty ones): a dict of
        lists, one per sequence, with an entry for each of its tokens but the first (with ``prefix``, ids before every sequence
        that are read once for all: for the first too): ``logprobs`` of the tokens, ``entropy`` of the distributions that they are
        drawn from, and with ``top`` the likeliest ``top_tokens`` and their ``top_logprobs`` (``ops.token_logprobs``).  Slots 0
        to ``len(sequences) - 1`` (the next one too with ``prefix``) hold new conversations afterwards."""
        self._check_prompts(sequences, prefix)
        self._check_new(sequences, prefix)
        V = self.model.cfg.vocab_size  # scores of no rows: what the settings are refused for
        ops.token_logprobs(torch.empty(0, V), torch.empty(0, dtype=torch.long), top=top, temperature=temperature)
        B, slots, first = len(sequences), list(range(len(sequences))), None
        if prefix is not None:
            first = self._read_prefix(prefix, B)
        h, _ = self._read(sequences, slots, prefix is None)
        # row t of a sequence answers for its token t + 1, the prefix's last row for the first ones
        rows, tokens, counts, at = [], [], [], 0
        for s in sequences:
            n = len(s)
            rows += ([-1] if first is not None else []) + list(range(at, at + n - 1))
            tokens += list(s if first is not None else s[1:])
            counts.append(len(tokens))
            at += n
        rows, tokens = torch.tensor(rows, dtype=torch.long).to(self.device), torch.tensor(tokens, dtype=torch.long).to(self.device)
        if first is not None:
            h = torch.cat([h, first])  # row -1
        step, parts = max(1, SCORE_LOGITS // V), []
        for a in range(0, max(1, len(rows)), step):
            logits = self._logits(h[rows[a:a + step]])
            parts.append([t.tolist() for t in ops.token_logprobs(logits, tokens[a:a + step], top=top, temperature=temperature)])
        self._check_waits()
        names = ("logprobs", "entropy", "top_tokens", "top_logprobs")[:len(parts[0])]
        flat = [sum(p, []) for p in zip(*parts)]
        return {name: [v[a:e] for a, e in zip([0] + counts[:-1], counts)] for name, v in zip(names, flat)}

    # ------------------------------------------------------------ generation
    @torch.no_grad()
    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int, temperature=1.0, top_k=0, top_p=1.0,
                 min_p=0.0, stop_token: Optional[int] = None, generator: Optional[torch.Generator] = None,
                 prefix: Optional[Sequence[int]] = None):
        """Answers to ``prompts`` (lists of token ids, at most ``max_sequences`` non-empty ones): returns
        ``(tokens, logprobs)``, one list per prompt, each at most ``max_new_tokens`` long and ending with
        ``stop_token`` where it was drawn.  The settings are numbers or one value per prompt;
        ``generator`` (on the model's device) makes the noise.  The prompts are new conversations in slots 0 to
        ``len(prompts) - 1``, which later hold every token that was run, those after a stop among them: conversations of
        ``prefill`` and ``step`` belong in other slots or another ``Generator``.  ``prefix`` (token ids) comes before every
        prompt and is read once for all, in slot ``len(prompts)``, where it stays."""
        B = len(prompts)
        self._check_prompts(prompts, prefix)
        if max_new_tokens < 1:
            return [[] for _ in prompts], [[] for _ in prompts]
        slots = list(range(B))
        V, dev = self.model.cfg.vocab_size, self.device
        row = lambda v, dt: torch.as_tensor(v, dtype=dt).expand(B).contiguous().to(dev)  # noqa: E731
        rules = (row(temperature, torch.float32), row(top_k, torch.int32), row(top_p, torch.float32), row(min_p, torch.float32))
        self._check_new(prompts, prefix)
        if prefix is not None:
            self._read_prefix(prefix, B)
        noise = lambda out: out.exponential_(generator=generator)  # noqa: E731
        t, lp = ops.sample(self.prefill(prompts, slots, fresh=prefix is None), noise(torch.empty(B, V, device=dev)), *rules)
        steps = [(t, lp)]
        done = (t < 0) | (t == stop_token) if stop_token is not None else t < 0
        replay = self.cuda_graph and max_new_tokens > 1 and self.state.on_device()
        if replay:
            graph, buf = self._graph_step(slots)
            for name, v in zip(("temperature", "top_k", "top_p", "min_p"), rules):
                buf[name].copy_(v)
            buf["tokens"].copy_(t.clamp(min=0))
        for i in range(1, max_new_tokens):
            if i % 16 == 0 and bool(done.all()):  # the host waits for the device every 16 tokens only
                break
            if replay:
                self.state.cut_back(self.state.check_room(slots, [1] * B))
                noise(buf["noise"])
                graph.replay()
                t, lp = (o.clone() for o in buf["out"])
                for s in slots:
                    self.state.lengths[s] += 1
                    self.state.rows[s] += 1
            else:
                t, lp = ops.sample(self.step(t.clamp(min=0), slots), noise(torch.empty(B, V, device=dev)), *rules)
            steps.append((t, lp))
            done = done | (t < 0) | (t == stop_token) if stop_token is not None else done | (t < 0)
        tokens = torch.stack([s[0] for s in steps], 1).tolist()
        logprobs = torch.stack([s[1] for s in steps], 1).tolist()
        self._check_waits()
        for ts, ls in zip(tokens, logprobs):
            end = next((i + (x >= 0) for i, x in enumerate(ts) if x < 0 or x == stop_token), len(ts))
            del ts[end:], ls[end:]
        return tokens, logprobs
