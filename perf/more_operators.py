"""Measured cases of the operators that keep, read and thin out an attention cache, and that score answers.

* ``ops.cached_attention`` -- the new tokens of several conversations rotated, written into the cache and
  answered from it; conversations that share a prefix read its rows once for all; on request every cached row
  gathers the attention that it gets;
* ``ops.cache_evict`` -- a conversation's cache thinned out to a number of rows, those that got least attention
  first, the newest ones kept;
* ``ops.token_logprobs`` -- log-probabilities of given tokens, the entropy of every row and its likeliest
  alternatives, with a backward pass.

``own = False`` runs them in plain torch operations in 32 bits, ``own = True`` as the framework
runs them."""
import math

import torch

own = False

DEV = "cuda"
CLIP = 1e3


# ----------------------------------------------------------------------------- cases
def listed():
    attn = dict(op="attn", heads=16, kv_heads=16, head=128, prefix=0, tracked=False)
    return [
        # one conversation being answered: one token through one attention layer of the reference run (6 heads)
        dict(attn, name="attn token x1", heads=6, kv_heads=6, lens="1x1", had="1000-1000"),
        # a serving batch, one token each, conversations of uneven length
        dict(attn, name="attn token x64", lens="64x1", had="60-2500"),
        # many answers under one long instruction: a shared prefix, short conversations of their own
        dict(attn, name="attn token x64 on a prefix", lens="64x1", had="1-500", prefix=8000),
        # a serving batch whose cache is thinned out later: rows gather attention; four query heads a key head
        dict(attn, name="attn tracked token x48", heads=32, kv_heads=8, lens="48x1", had="200-4000", tracked=True),
        # one long document read from its start
        dict(attn, name="attn long prompt", lens="1x8192", had="0-0"),
        # several questions of uneven length about one document, checked in one go
        dict(attn, name="attn questions on a prefix", lens="700,17,1,333,64,1025,255,12", had="0-0", prefix=4100),
        # one conversation of the reference run's layer, cut to its budget
        dict(op="evict", name="evict x1", convs=1, kv_heads=6, head=128, keep=1024, over=128, recent=64),
        # a serving batch of grown conversations, cut to half
        dict(op="evict", name="evict x64", convs=64, kv_heads=16, head=128, keep=512, over=512, recent=128),
        # a drawn token's score and its alternatives, for a serving batch
        dict(op="score", name="score x64", rows=64, vocab=50304, dtype="bf16", top=5, grad=False),
        # scoring long answers with alternatives, the reference run's vocabulary
        dict(op="score", name="score x2048", rows=2048, vocab=128256, dtype="bf16", top=8, grad=False),
        # a training step on the answers' log-probabilities with an entropy bonus
        dict(op="score", name="score gradient x4096", rows=4096, vocab=50304, dtype="bf16", top=0, grad=True),
        # the same from logits in 32 bits, the reference's default vocabulary
        dict(op="score", name="score gradient fp32", rows=300, vocab=151936, dtype="fp32", top=0, grad=True),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("attn", "attn", "attn", "evict", "score", "score"))
    if op == "attn":
        head = rng.choice((128, 128, 64, 96))
        kv = _log(rng, 1, 16)
        heads = kv * rng.choice((1, 1, 2, 4, 3))
        kind = rng.choice(("token", "token", "drafts", "prompts"))
        prefix = rng.choice((0, 0, _log(rng, 1, 8000)))
        if kind == "token":
            n, lo = _log(rng, 1, 64), _log(rng, 1, 500)
            return dict(op=op, heads=heads, kv_heads=kv, head=head, lens="%dx1" % n, had="%d-%d" % (lo, _log(rng, lo, 2500)),
                        prefix=prefix, tracked=rng.random() < 0.3)
        if kind == "drafts":
            n = _log(rng, 1, 32)
            return dict(op=op, heads=heads, kv_heads=kv, head=head, lens=",".join(str(_log(rng, 1, 12)) for _ in range(n)),
                        had="0-%d" % _log(rng, 1, 2000), prefix=prefix, tracked=rng.random() < 0.3)
        n = _log(rng, 1, 12)
        lens = [_log(rng, 1, 4000 // n) for _ in range(n)]
        kv = min(kv, 16 // (heads // kv))
        heads = min(heads, 16) // kv * kv
        return dict(op=op, heads=heads, kv_heads=kv, head=head, lens=",".join(map(str, lens)), had="0-%d" % _log(rng, 1, 1000),
                    prefix=min(prefix, 4000), tracked=rng.random() < 0.3)
    if op == "evict":
        keep = _log(rng, 32, 1024)
        return dict(op=op, convs=_log(rng, 1, 48), kv_heads=_log(rng, 1, 16), head=rng.choice((128, 64, 96)), keep=keep,
                    over=_log(rng, 1, 600), recent=rng.randrange(0, keep))
    grad = rng.random() < 0.5
    vocab = rng.choice((4096, 50304, 128256, 151936, _log(rng, 300, 150000)))
    rows = _log(rng, 1, max(1, 150_000_000 // vocab if grad else 200_000_000 // vocab))
    return dict(op=op, rows=min(rows, 4096), vocab=vocab, dtype=rng.choice(("bf16", "bf16", "fp32")),
                top=0 if grad else rng.choice((0, 1, 5, 20)), grad=grad)


def _lens(case):
    text = case["lens"]
    if "x" in text:
        n, l = text.split("x")
        return [int(l)] * int(n)
    return [int(l) for l in text.split(",")]


def _had(case):
    """The rows that each conversation has in the cache already, spread over the case's range."""
    lo, hi = map(int, case["had"].split("-"))
    return [lo + (i * 2654435761 + 12345) % (1 << 32) * (hi - lo) // ((1 << 32) - 1) for i in range(len(_lens(case)))]


def _dtype(case):
    return torch.float32 if case.get("dtype") == "fp32" else torch.bfloat16


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = _dtype(case)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=dtype) * std

    def permuted(n):
        return torch.randperm(n, generator=gen, device=DEV)

    s = {"case": case}
    if case["op"] == "score":
        R, V = case["rows"], case["vocab"]
        # a language model's logits: a broad bulk and a handful of likely tokens in every row
        logits = normal(R, V, std=2.0, dtype=dt)
        top = torch.randint(0, V, (R, 12), generator=gen, device=DEV)
        logits.scatter_add_(1, top, (torch.rand(R, 12, generator=gen, device=DEV) * 8 + 4).to(dt))
        s["tokens"] = torch.where(torch.rand(R, generator=gen, device=DEV) < 0.7, top[:, 0],
                                  torch.randint(0, V, (R,), generator=gen, device=DEV))
        if case["grad"]:
            s["tokens"] = torch.where(torch.rand(R, generator=gen, device=DEV) < 0.1, -100, s["tokens"])  # prompts' rows
            s["weights"] = (normal(R), normal(R, std=0.01))  # the losses' gradients of logprobs and entropies
        else:
            logits[:, V // 3: V // 3 + V // 8] = float("-inf")  # tokens that a grammar forbids
        s["logits"] = logits.requires_grad_(case["grad"])
        return s
    Hk, D = case["kv_heads"], case["head"]
    if case["op"] == "evict":
        B, keep, over = case["convs"], case["keep"], case["over"]
        n, pool, M = keep + over, case["convs"] + 2, case["keep"] + case["over"] + 5
        s["slots"] = permuted(pool)[:B].to(torch.int32)
        s.update(k_cache=normal(pool, Hk, M, D, dtype=dt), v_cache=normal(pool, Hk, M, D, dtype=dt))
        s["lengths"] = torch.full((pool,), n, dtype=torch.int32, device=DEV)
        s["seen"] = torch.full((pool,), n + 700, dtype=torch.int32, device=DEV)
        # heavy-tailed sums; the tokens since the last cut lie behind the rows that it kept
        s["gathered"] = torch.exp(normal(pool, Hk, M, std=1.5))
        old = torch.rand(pool, Hk, keep + 700, generator=gen, device=DEV).argsort(-1)[..., :keep]
        new = torch.arange(keep + 700, M + 700, device=DEV).expand(pool, Hk, -1)
        s["positions"] = torch.cat([old, new], -1).to(torch.int32)
        s.update(mass=s["gathered"].clone(), held=s["positions"].clone())
        return s
    lens, had, H, P = _lens(case), _had(case), case["heads"], case["prefix"]
    B, T = len(lens), sum(lens)
    pool = B + 3
    M = max(max(h + n for h, n in zip(had, lens)), P) + 5
    order = permuted(pool)
    s["slots"] = order[:B].to(torch.int32)
    s["one"] = all(n == 1 for n in lens)
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens, dtype=torch.int32), 0)
    s["cu"] = cu.to(DEV)
    s["lengths"] = torch.zeros(pool, dtype=torch.int32, device=DEV)
    s["lengths"][order[:B]] = torch.tensor(had, dtype=torch.int32, device=DEV)
    s["prefix"] = None
    if P:
        s["prefix"] = order[B].to(torch.int32).expand(B).contiguous()
        s["lengths"][order[B]] = P
    s["seen"] = s["lengths"] + P
    angle = torch.arange(P + M, device=DEV)[:, None].double() / 10000 ** (torch.arange(0, D, 2, device=DEV).double() / D)
    angle = torch.cat([angle, angle], -1)
    s.update(cos=angle.cos().float(), sin=angle.sin().float())
    qkv = normal(T, (H + 2 * Hk) * D, dtype=dt)  # one projection's output: queries, keys and values side by side
    qkv[:, :H * D] *= 1.5
    s.update(q=qkv[:, :H * D], k=qkv[:, H * D:(H + Hk) * D], v=qkv[:, (H + Hk) * D:])
    s.update(k_cache=normal(pool, Hk, M, D, dtype=dt), v_cache=normal(pool, Hk, M, D, dtype=dt), mass=None, held=None)
    if case["tracked"]:
        s["mass"] = torch.exp(normal(pool, Hk, M))
        s["held"] = torch.arange(M, device=DEV, dtype=torch.int32).expand(pool, Hk, M).contiguous()
    return s


# ----------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    from atomic_ai_hybrid_b200 import ops

    case = s["case"]
    if case["op"] == "score":
        out = ops.token_logprobs(s["logits"], s["tokens"], top=case["top"])
        named = dict(zip(("logprobs", "entropy", "top_tokens", "top_logprobs"), out))
        if case["grad"]:
            named["gradient"] = torch.autograd.grad(out, [s["logits"]], list(s["weights"]))[0]
            named = {n: t.detach() for n, t in named.items()}
        return named
    if case["op"] == "evict":
        s["mass"].copy_(s["gathered"])  # what the layers gathered since the last cut
        s["held"].copy_(s["positions"])
        ops.cache_evict(s["k_cache"], s["v_cache"], s["mass"], s["held"], s["lengths"], s["seen"], case["keep"],
                        recent=case["recent"], slots=s["slots"])
        return {n: s[n] for n in ("k_cache", "v_cache", "mass", "held")}
    cu = None if s["one"] else s["cu"]  # without offsets every row is one token of its own sequence
    o = ops.cached_attention(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["lengths"], cos=s["cos"], sin=s["sin"],
                             cu_seqlens=cu, slots=s["slots"], prefix=s["prefix"], seen=s["seen"], mass=s["mass"],
                             held=s["held"])
    out = {"o": o, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["tracked"]:
        out.update(mass=s["mass"], held=s["held"])
    return out


# ----------------------------------------------------------------------------- plain forms
def _clip(x):
    return torch.nan_to_num(x.clamp(-CLIP, CLIP), nan=0.0)


def _rotated(x, at, cos, sin):
    a, b = x.chunk(2, -1)
    return x * cos[at][:, None] + torch.cat([-b, a], -1) * sin[at][:, None]


def _plain_attn(s):
    case = s["case"]
    lens, had, P = _lens(case), _had(case), case["prefix"]
    H, Hk, D = case["heads"], case["kv_heads"], case["head"]
    G, T, scale = H // Hk, sum(lens), 1.0 / math.sqrt(D)
    slots = s["slots"].long()
    who = torch.repeat_interleave(torch.arange(len(lens), device=DEV), (s["cu"][1:] - s["cu"][:-1]).long(), output_size=T)
    nth = torch.arange(T, device=DEV) - s["cu"][:-1].long()[who]
    row, at, slot = s["lengths"].long()[slots][who] + nth, s["seen"].long()[slots][who] + nth, slots[who]
    q = _clip(_rotated(s["q"].float().view(T, H, D), at, s["cos"], s["sin"]))
    k = _clip(_rotated(s["k"].float().view(T, Hk, D), at, s["cos"], s["sin"]))
    s["k_cache"][slot, :, row] = k.to(s["k_cache"].dtype)
    s["v_cache"][slot, :, row] = _clip(s["v"].float()).view(T, Hk, D).to(s["v_cache"].dtype)
    if case["tracked"]:
        s["mass"][slot, :, row] = 0.0
        s["held"][slot, :, row] = at.to(torch.int32)[:, None]
    q = q.view(T, Hk, G, D).transpose(0, 1)  # queries by key head
    o = torch.empty(Hk, T, G, D, device=DEV)
    if P:  # the shared rows once for all
        shared = s["prefix"][0].long()
        kp, vp = s["k_cache"][shared, :, :P].float(), s["v_cache"][shared, :, :P].float()
    for i, (n, h) in enumerate(zip(lens, had)):
        first, slot = sum(lens[:i]), slots[i]
        ki, vi = s["k_cache"][slot, :, :h + n].float(), s["v_cache"][slot, :, :h + n].float()
        step = max(1, min(n, (1 << 28) // ((h + n + P) * H)))
        for t in range(0, n, step):
            e = min(n, t + step)
            qi = q[:, first + t:first + e].reshape(Hk, -1, D) * scale
            w = qi @ ki.transpose(1, 2)
            seen = torch.arange(h + n, device=DEV) <= torch.arange(h + t, h + e, device=DEV)[:, None]
            w = torch.where(seen.repeat_interleave(G, 0), w, torch.full((), float("-inf"), device=DEV))
            top = w.max(-1, keepdim=True).values
            if P:
                wp = qi @ kp.transpose(1, 2)
                top = torch.maximum(top, wp.max(-1, keepdim=True).values)
                wp = torch.exp(wp - top)
            w = torch.exp(w - top)
            total = w.sum(-1, keepdim=True)
            y = w @ vi
            if P:
                total = total + wp.sum(-1, keepdim=True)
                y = y + wp @ vp
            o[:, first + t:first + e] = (y / total).view(Hk, e - t, G, D)
            if case["tracked"]:
                s["mass"][slot, :, :h + n] += (w / total).sum(1)
    out = {"o": o.transpose(0, 1).reshape(T, H * D).to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["tracked"]:
        out.update(mass=s["mass"], held=s["held"])
    return out


def _plain_evict(s):
    case = s["case"]
    keep, recent, n = case["keep"], case["recent"], case["keep"] + case["over"]
    s["mass"].copy_(s["gathered"])
    s["held"].copy_(s["positions"])
    slots = s["slots"].long()
    mass, held = s["mass"][slots, :, :n], s["held"][slots, :, :n]
    newest = held >= (s["seen"][slots] - recent)[:, None, None]
    rank = torch.where(newest, torch.full((), float("inf"), device=DEV), mass)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros(rank.shape, dtype=torch.bool, device=DEV).scatter_(-1, order[..., :keep], True)
    b, h, hole = torch.nonzero(~kept[..., :keep], as_tuple=True)  # in rows' order, as many as kept rows lie behind
    row = torch.nonzero(kept[..., keep:], as_tuple=True)[2] + keep
    for name in ("k_cache", "v_cache", "mass", "held"):
        s[name][slots[b], h, hole] = s[name][slots[b], h, row]
    return {name: s[name] for name in ("k_cache", "v_cache", "mass", "held")}


def _plain_score(s):
    case = s["case"]
    R, V = case["rows"], case["vocab"]
    out = {n: [] for n in ("logprobs", "entropy", "top_tokens", "top_logprobs", "gradient")}
    step = max(1, (1 << 28) // V)
    for r in range(0, R, step):
        x, y = s["logits"].detach()[r:r + step].float(), s["tokens"][r:r + step]
        d = x - x.max(1, keepdim=True).values
        e = torch.exp(d)
        total = e.sum(1, keepdim=True)
        p, logp = e / total, d - torch.log(total)
        given = y >= 0
        out["logprobs"].append(torch.where(given, logp.gather(1, y.clamp(min=0)[:, None])[:, 0], torch.zeros((), device=DEV)))
        logp = torch.where(p > 0, logp, torch.zeros((), device=DEV))
        entropy = -(p * logp).sum(1)
        out["entropy"].append(entropy)
        if case["top"]:
            best, index = torch.sort(x, dim=1, descending=True, stable=True)  # ties: lowest index first
            out["top_tokens"].append(index[:, :case["top"]].clone())
            out["top_logprobs"].append((best - best[:, :1] - torch.log(total))[:, :case["top"]].clone())
        if case["grad"]:
            g, ge = (w[r:r + step] for w in s["weights"])
            g = g * given
            dx = -p * (g + ge * entropy)[:, None] - p * logp * ge[:, None]
            dx.scatter_add_(1, y.clamp(min=0)[:, None], g[:, None])
            out["gradient"].append(dx.to(s["logits"].dtype))
    return {n: torch.cat(ts) for n, ts in out.items() if ts}


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "evict": _plain_evict, "score": _plain_score}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------- work
def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] == "score":
        n, R = case["rows"] * case["vocab"], case["rows"]
        return {"bytes": n * size * (2 if case["grad"] else 1) + R * (8 + 8 + 12 * case["top"]),
                "flops": n * (12 if case["grad"] else 6)}
    Hk, D = case["kv_heads"], case["head"]
    if case["op"] == "evict":
        keep, over, recent = case["keep"], case["over"], case["recent"]
        rest, late = keep + over - recent, min(recent, over)  # the newest stay; of the others, any as likely as another
        moved = late + (over - late) * (keep - recent) / rest
        # per head the sums and positions looked at (and set anew before), the moved rows read and written
        return {"bytes": case["convs"] * Hk * (8 * (keep + over) + moved * (2 * 2 * D * size + 16)),
                "flops": case["convs"] * Hk * (keep + over)}
    lens, had, P, H = _lens(case), _had(case), case["prefix"], case["heads"]
    T, rows = sum(lens), sum(had) + P
    pairs = sum(n * (h + P) + n * (n + 1) // 2 for n, h in zip(lens, had))
    return {"bytes": size * D * (2 * T * H + 4 * T * Hk + 2 * rows * Hk) + (8 * Hk * (sum(had) + T) if case["tracked"] else 0),
            "flops": 4 * D * H * pairs}


# ----------------------------------------------------------------------------- 64 bits
def _exact_attn(s):
    case = s["case"]
    lens, had, P = _lens(case), _had(case), case["prefix"]
    H, Hk, D = case["heads"], case["kv_heads"], case["head"]
    G = H // Hk
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    mass = None if s["mass"] is None else s["mass"].double()
    held = None if s["held"] is None else s["held"].clone()
    slots = s["slots"].tolist()
    half, out, at = D // 2, [], 0
    for n, h, slot in zip(lens, had, slots):
        c, sn = (s[name][P + h:P + h + n, :half].double()[:, None] for name in ("cos", "sin"))

        def turned(x):
            x1, x2 = x[..., :half], x[..., half:]
            return torch.cat([x1 * c - x2 * sn, x2 * c + x1 * sn], -1).clamp(-CLIP, CLIP)

        q = turned(s["q"][at:at + n].double().view(n, H, D)).transpose(0, 1)
        k = turned(s["k"][at:at + n].double().view(n, Hk, D)).transpose(0, 1)
        kc[slot, :, h:h + n] = k
        vc[slot, :, h:h + n] = s["v"][at:at + n].double().view(n, Hk, D).transpose(0, 1).clamp(-CLIP, CLIP)
        stored = k.to(s["k_cache"].dtype).double()  # the attention reads the cache as it is kept
        keys, values = [kc[slot, :, :h], stored], [vc[slot, :, :h + n]]
        if P:
            shared = int(s["prefix"][0])
            keys, values = [kc[shared, :, :P]] + keys, [vc[shared, :, :P]] + values
        keys, values = torch.cat(keys, 1), torch.cat(values, 1)
        if mass is not None:
            mass[slot, :, h:h + n] = 0
            held[slot, :, h:h + n] = torch.arange(P + h, P + h + n, device=DEV, dtype=torch.int32)
        hidden = torch.ones(n, P + h + n, dtype=torch.bool, device=DEV).triu(P + h + 1)
        ys = []
        for j in range(H):
            w = torch.softmax((q[j] @ keys[j // G].t() / math.sqrt(D)).masked_fill(hidden, float("-inf")), -1)
            ys.append(w @ values[j // G])
            if mass is not None:
                mass[slot, j // G, :h + n] += w.sum(0)[P:]
        out.append(torch.stack(ys, 1).reshape(n, H * D))
        at += n
    named = {"o": torch.cat(out), "k_cache": kc, "v_cache": vc}
    if mass is not None:
        named.update(mass=mass, held=held)
    return named


def _exact_evict(s):
    case = s["case"]
    keep, recent, n = case["keep"], case["recent"], case["keep"] + case["over"]
    sums, positions, seen = s["gathered"].double().cpu(), s["positions"].cpu(), s["seen"].tolist()
    out = {"k_cache": s["k_cache"].clone(), "v_cache": s["v_cache"].clone(), "mass": s["gathered"].clone(),
           "held": s["positions"].clone()}
    for slot in s["slots"].tolist():
        for h in range(case["kv_heads"]):
            m, p = sums[slot, h, :n].tolist(), positions[slot, h, :n].tolist()
            best = sorted(range(n), key=lambda i: (p[i] < seen[slot] - recent, 0.0 if p[i] >= seen[slot] - recent else -m[i], i))
            kept = set(best[:keep])
            holes = torch.tensor([i for i in range(keep) if i not in kept], dtype=torch.long, device=DEV)
            rows = torch.tensor([i for i in range(keep, n) if i in kept], dtype=torch.long, device=DEV)
            for t in out.values():
                t[slot, h, holes] = t[slot, h, rows]
    return {name: t if name == "held" else t.double() for name, t in out.items()}


def _exact_score(s):
    case = s["case"]
    out = {n: [] for n in ("logprobs", "entropy", "top_tokens", "top_logprobs", "gradient")}
    for r in range(0, case["rows"], 256):
        x, y = s["logits"].detach()[r:r + 256].double(), s["tokens"][r:r + 256]
        logp = torch.log_softmax(x, 1)
        p = logp.exp()
        shift = -torch.xlogy(p, p)
        entropy = shift.sum(1)
        got = logp.gather(1, y.clamp(min=0)[:, None])[:, 0]
        out["logprobs"].append(torch.where(y < 0, 0.0, got))
        out["entropy"].append(entropy)
        if case["top"]:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            out["top_tokens"].append(order)
            out["top_logprobs"].append(logp.gather(1, order))
        if case["grad"]:
            g, ge = (w[r:r + 256].double()[:, None] for w in s["weights"])
            onehot = torch.zeros_like(p).scatter_(1, y.clamp(min=0)[:, None], 1.0)
            out["gradient"].append(torch.where(y[:, None] < 0, 0.0, g) * (onehot - p) + ge * (shift - p * entropy[:, None]))
    return {n: torch.cat(ts) for n, ts in out.items() if ts}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "evict": _exact_evict, "score": _exact_score}[case["op"]](s)
