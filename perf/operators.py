"""Measured cases of the operators that answer from a trained hybrid model.

Three operators, each updating the recurrent state of its layer in place where it has one:

* ``ops.selective_scan`` -- Mamba2's short causal convolution and per-channel-dt scan, for prompts
  (packed or padded, from any state) and for single tokens;
* ``ops.gdn2_recurrent`` -- GDN-2's convolutions, gates and delta rule for one or a few tokens;
* ``ops.sample`` -- the next token from logits and given exponential noise, with temperature,
  top-k, top-p and min-p per row.

``own = False`` runs them in plain torch operations in 32 bits, ``own = True`` as the framework
runs them."""
import torch

own = False

DEV = "cuda"
TAPS = 4
NEG_DA = -20.0


# ----------------------------------------------------------------------------- cases
def listed():
    scan = dict(op="scan", headdim=64, state=128, dtype="bf16")
    gdn = dict(op="gdn", head=128, dtype="bf16")
    return [
        # one conversation being answered: one token through one Mamba2 layer of hybrid_1b
        dict(scan, name="scan token x1", channels=2048, lens="1x1"),
        # a serving batch: one token for each of 64 conversations
        dict(scan, name="scan token x64", channels=2048, lens="64x1"),
        # the reference run's Mamba2 layer (1536 channels in 8 heads), activations in 32 bits
        dict(scan, name="scan token x200 fp32", channels=1536, headdim=192, lens="200x1", dtype="fp32"),
        # several prompts of uneven lengths packed one after another, a one-token one among them
        dict(scan, name="scan ragged prompts", channels=2048, lens="700,17,1,333,64,1025,255"),
        # one long document
        dict(scan, name="scan one long prompt", channels=2048, lens="1x8192"),
        # a batch of prompts through a layer of hybrid_long
        dict(scan, name="scan prompt batch", channels=4096, lens="8x2048"),
        # one conversation being answered: one token through one GDN-2 layer of hybrid_1b
        dict(gdn, name="gdn token x1", heads=16, lens="1x1"),
        # a serving batch
        dict(gdn, name="gdn token x128", heads=16, lens="128x1"),
        # checking a few drafted tokens of several conversations at once (the reference run's layer)
        dict(gdn, name="gdn drafts", heads=6, lens="5,8,1,3,5,5,7,2,5,5,5,4,6,5,5,1"),
        # one conversation, the reference's default vocabulary
        dict(op="sample", name="sample x1", rows=1, vocab=151936, dtype="bf16", rules="mixed"),
        # a serving batch, hybrid_1b's vocabulary, every row with its own settings
        dict(op="sample", name="sample x64", rows=64, vocab=50304, dtype="bf16", rules="mixed"),
        # a large batch from logits in 32 bits, the reference run's vocabulary
        dict(op="sample", name="sample x256 fp32", rows=256, vocab=128256, dtype="fp32", rules="nucleus"),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("scan", "scan", "gdn", "sample"))
    if op == "scan":
        state, headdim = rng.choice(((128, 64), (128, 64), (64, 64), (128, 192), (32, 64)))
        channels = headdim * _log(rng, 2, 4096 // headdim)
        kind = rng.choice(("token", "prompts", "prompts"))
        if kind == "token":
            return dict(op=op, channels=channels, headdim=headdim, state=state, lens="%dx1" % _log(rng, 1, 200),
                        dtype=rng.choice(("bf16", "bf16", "fp32")))
        n, most = _log(rng, 1, 16), 16384
        lens = [_log(rng, 1, most // n) for _ in range(n)]
        return dict(op=op, channels=channels, headdim=headdim, state=state, lens=",".join(map(str, lens)), dtype="bf16")
    if op == "gdn":
        head = rng.choice((128, 128, 64, 96))
        heads = _log(rng, 2, 24)
        n = _log(rng, 1, 128)
        if rng.random() < 0.5:
            lens = "%dx1" % n
        else:
            lens = ",".join(str(_log(rng, 1, 12)) for _ in range(min(n, 32)))
        return dict(op=op, heads=heads, head=head, lens=lens, dtype="bf16")
    vocab = rng.choice((4096, 50304, 128256, 151936, _log(rng, 300, 150000)))
    return dict(op=op, rows=_log(rng, 1, 256), vocab=vocab, dtype=rng.choice(("bf16", "fp32")),
                rules=rng.choice(("mixed", "nucleus", "topk", "open")))


def _lens(case):
    text = case["lens"]
    if "x" in text:
        n, l = text.split("x")
        return [int(l)] * int(n)
    return [int(l) for l in text.split(",")]


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = _dtype(case)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device=DEV) * std + mean

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=gen, device=DEV) * (hi - lo) + lo

    s = {"case": case}
    if case["op"] == "sample":
        B, V = case["rows"], case["vocab"]
        # a language model's logits: a broad bulk and a handful of likely tokens in every row
        logits = normal(B, V, std=2.0)
        top = torch.randint(0, V, (B, 12), generator=gen, device=DEV)
        logits.scatter_add_(1, top, uniform(4.0, 12.0, B, 12))
        if case["rules"] != "open":  # tokens that a grammar forbids
            logits[:, V // 3: V // 3 + V // 8] = float("-inf")
        s["logits"] = logits.to(dt)
        s["noise"] = torch.empty(B, V, device=DEV).exponential_(generator=gen)
        one = torch.ones(B, device=DEV)
        zero = torch.zeros(B, dtype=torch.int32, device=DEV)
        s.update(temperature=one, top_k=zero, top_p=one, min_p=0 * one)
        row = torch.arange(B, device=DEV)
        if case["rules"] in ("mixed", "topk", "nucleus"):
            s["temperature"] = uniform(0.6, 1.3, B)
        if case["rules"] in ("mixed", "topk"):
            s["top_k"] = torch.randint(2, 200, (B,), generator=gen, device=DEV, dtype=torch.int32)
        if case["rules"] in ("mixed", "nucleus"):
            s["top_p"] = uniform(0.7, 0.98, B)
        if case["rules"] == "mixed" and B > 1:
            s["temperature"] = torch.where(row % 8 == 3, 0.0, s["temperature"])  # greedy rows
            s["top_k"] = torch.where(row % 4 == 1, 0, s["top_k"]).to(torch.int32)
            s["min_p"] = torch.where(row % 4 == 2, 0.05, 0.0).to(torch.float32)
        return s

    lens = _lens(case)
    B, T = len(lens), sum(lens)
    pool = B + 3  # the layer's state pool has other conversations' slots too
    s["slots"] = torch.randperm(pool, generator=gen, device=DEV)[:B].to(torch.int32)
    s["one"] = all(l == 1 for l in lens)
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens, dtype=torch.int32), 0)
    s["cu"] = cu.to(DEV)
    if case["op"] == "scan":
        C, P, N = case["channels"], case["headdim"], case["state"]
        H = C // P
        xz = normal(T, 2 * C).to(dt)  # in_proj's output: the scan's input and its gate side by side
        step = uniform(1e-3, 0.1, C)
        bias = step + torch.log(-torch.expm1(-step))
        s.update(x=xz[:, :C], dt=(normal(T, C, std=0.7) + bias).to(dt), A=-uniform(1.0, 16.0, H),
                 B=normal(T, N).to(dt), C=normal(T, N).to(dt),
                 conv_w=normal(C, TAPS, std=0.4), conv_b=normal(C, std=0.1),
                 conv_state=normal(pool, TAPS - 1, C).to(dt), state=normal(pool, H, P, N, std=0.3))
        return s
    H, D = case["heads"], case["head"]
    d = H * D
    s.update(x=[normal(T, d).to(dt) for _ in range(3)], gates=[normal(T, d).to(dt) for _ in range(3)],
             conv_w=[normal(d, TAPS, std=0.4).to(dt) for _ in range(3)], conv_b=[normal(d, std=0.1) for _ in range(3)],
             decay_a=normal(H, std=0.5, mean=-1.0),
             conv_state=normal(pool, 3, TAPS - 1, d).to(dt), state=normal(pool, H, D, D, std=0.1))
    return s


# ----------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    from atomic_ai_hybrid_b200 import ops

    case = s["case"]
    if case["op"] == "sample":
        tokens, logprobs = ops.sample(s["logits"], s["noise"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return {"tokens": tokens, "logprobs": logprobs}
    cu = None if s["one"] else s["cu"]  # without offsets every row is one token of its own sequence
    if case["op"] == "scan":
        y = ops.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["conv_w"], s["conv_b"], s["conv_state"],
                               s["state"], cu_seqlens=cu, slots=s["slots"])
    else:
        y = ops.gdn2_recurrent(*s["x"], *s["gates"], s["conv_w"], s["conv_b"], s["decay_a"], s["conv_state"],
                               s["state"], cu_seqlens=cu, slots=s["slots"])
    return {"y": y, "conv_state": s["conv_state"], "state": s["state"]}


# ----------------------------------------------------------------------------- plain forms
def _sanitize(x, c):
    return torch.nan_to_num(x.clamp(-c, c), nan=0.0, posinf=c, neginf=-c)


def _softplus(x):
    return torch.where(x > 20.0, x, torch.log1p(torch.exp(torch.clamp(x, max=20.0))))


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _padded(s, lens):
    """Rows of the packed tokens as a (sequences, longest) table, and where the table has a token."""
    B, Lm = len(lens), max(lens)
    start = s["cu"][:-1].long()
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    at = torch.arange(Lm, device=DEV)
    has = at[None] < n[:, None]
    row = torch.where(has, start[:, None] + at[None], torch.zeros_like(start)[:, None])
    return row, has, n


def _conv(x, has, row, window, w, b):
    """Causal convolution over a window of three earlier tokens and the table's, and the new window."""
    n = has.sum(1)
    ext = torch.cat([window.float(), x.float()[row] * has[..., None]], 1)
    L = row.shape[1]
    w = w.float()
    y = ext[:, 0:L] * w[:, 0] + ext[:, 1:L + 1] * w[:, 1] + ext[:, 2:L + 2] * w[:, 2] + ext[:, 3:L + 3] * w[:, 3]
    last = ext.gather(1, (n[:, None] + torch.arange(TAPS - 1, device=DEV))[..., None].expand(-1, -1, ext.shape[2]))
    return _silu(y + b.float()), last


def _plain_scan(s, chunk=32):
    case = s["case"]
    lens = _lens(case)
    C, P, N = case["channels"], case["headdim"], case["state"]
    H, slots = C // P, s["slots"].long()
    row, has, _ = _padded(s, lens)
    B, L = row.shape
    x, window = _conv(s["x"], has, row, s["conv_state"][slots], s["conv_w"], s["conv_b"])
    x = _sanitize(x, 1e3)
    dt = _softplus(s["dt"].float()).clamp(1e-2, 1.0)[row] * has[..., None]
    Bm = _sanitize(s["B"].float(), 1e3)[row] * has[..., None]
    Cm = _sanitize(s["C"].float(), 1e3)[row]
    dA = (dt * s["A"].repeat_interleave(P)).clamp(min=NEG_DA)
    u = dt * x
    S = s["state"][slots].reshape(B, C, N)
    ys = []
    for t in range(0, L, chunk):  # the state goes from chunk to chunk, tokens within one are joined at once
        e = min(L, t + chunk)
        cum = torch.cumsum(dA[:, t:e], 1)
        m = e - t
        low = torch.ones(m, m, device=DEV, dtype=torch.bool).tril()
        decay = torch.exp(torch.where(low[None, :, :, None], cum[:, :, None] - cum[:, None], torch.full((), -1e4, device=DEV)))
        CB = Cm[:, t:e] @ Bm[:, t:e].transpose(1, 2)
        y = (decay * CB[..., None] * u[:, None, t:e]).sum(2)
        ys.append(y + torch.exp(cum) * (Cm[:, t:e] @ S.transpose(1, 2)))
        to_end = torch.exp(cum[:, -1:] - cum) * u[:, t:e]
        S = S * torch.exp(cum[:, -1])[..., None] + to_end.transpose(1, 2) @ Bm[:, t:e]
    y = torch.cat(ys, 1)[has]
    s["conv_state"][slots] = window.to(s["conv_state"].dtype)
    s["state"][slots] = S.view(B, H, P, N)
    return {"y": y.to(s["x"].dtype), "conv_state": s["conv_state"], "state": s["state"]}


def _plain_gdn(s):
    case = s["case"]
    lens = _lens(case)
    H, D = case["heads"], case["head"]
    slots = s["slots"].long()
    row, has, n = _padded(s, lens)
    B, L = row.shape
    qkv, windows = zip(*[_conv(x, has, row, s["conv_state"][slots, i], w, b)
                         for i, (x, w, b) in enumerate(zip(s["x"], s["conv_w"], s["conv_b"]))])
    q, k, v = (t.view(B, L, H, D) for t in qkv)
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-12)
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-12)
    v = v.clamp(-50.0, 50.0)
    b, w, f = (t.float()[row].view(B, L, H, D) for t in s["gates"])
    b, w = 1.0 / (1.0 + torch.exp(-b)), 1.0 / (1.0 + torch.exp(-w))
    g = -torch.exp(s["decay_a"].clamp(-20.0, 20.0))[:, None] * _softplus(f)
    alpha = torch.exp(torch.nan_to_num(g, nan=0.0).clamp(-1e3, 0.0))
    live = has[..., None, None]
    alpha = torch.where(live, alpha, torch.ones_like(alpha))
    k, bk, wv = k * live, b * k * live, w * v * live
    h = s["state"][slots]
    outs = []
    for t in range(L):  # the delta rule goes token by token
        h = h * alpha[:, t, :, :, None]
        new = wv[:, t] - (bk[:, t, :, None] @ h)[:, :, 0]
        h = h + k[:, t, :, :, None] * new[:, :, None]
        outs.append((q[:, t, :, None] @ h)[:, :, 0])
    o = torch.stack(outs, 1).reshape(B, L, H * D)[has]
    s["conv_state"][slots] = torch.stack(windows, 1).to(s["conv_state"].dtype)
    s["state"][slots] = h
    return {"y": o.to(s["x"][0].dtype), "conv_state": s["conv_state"], "state": s["state"]}


def _plain_sample(s):
    logits = s["logits"].float()
    B, V = logits.shape
    T = s["temperature"][:, None]
    greedy = T == 0.0
    k = torch.where(greedy, 1, torch.where(s["top_k"][:, None] <= 0, V, s["top_k"][:, None]))
    T = torch.where(greedy, 1.0, T)
    d, index = torch.sort(logits, dim=1, descending=True, stable=True)  # ties: lowest index first
    d = (d[:, :1] - d) / T
    mass = torch.exp(-d)
    cum = torch.cumsum(mass, 1)
    total = cum[:, -1:]
    rank = torch.arange(V, device=logits.device)[None]
    kept = (rank < k) & ((cum - mass < s["top_p"][:, None] * total) | (rank == 0)) & (mass >= s["min_p"][:, None]) & (mass > 0)
    score = -d - torch.log(s["noise"].gather(1, index))
    score = torch.where(kept, score, torch.full((), float("-inf"), device=score.device))
    best = score.max(1, keepdim=True).values
    tokens = torch.where(score == best, index, V).min(1, keepdim=True).values
    dl = (logits.max(1, keepdim=True).values - logits.gather(1, tokens)) / T
    return {"tokens": tokens[:, 0], "logprobs": (-dl - torch.log(total))[:, 0]}


def run(state):
    if own:
        return _run_own(state)
    return {"scan": _plain_scan, "gdn": _plain_gdn, "sample": _plain_sample}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------- work
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (size + 4) + case["rows"] * (4 * 4 + 8 + 4), "flops": 6 * n}
    lens = _lens(case)
    B, T = len(lens), sum(lens)
    if case["op"] == "scan":
        C, N = case["channels"], case["state"]
        return {"bytes": size * T * (3 * C + 2 * N) + B * C * (8 * N + 2 * 3 * size) + C * (4 * TAPS + 4),
                "flops": T * C * (5 * N + 2 * TAPS + 12)}
    H, D = case["heads"], case["head"]
    d = H * D
    return {"bytes": size * T * 7 * d + B * (8 * H * D * D + 2 * 9 * d * size) + 3 * d * (TAPS * size + 4),
            "flops": T * H * D * (7 * D + 60)}


# ----------------------------------------------------------------------------- 64 bits
def _window64(x, state, w, b, lens, slots):
    """SiLU of the convolution, sequence by sequence, and the pool of windows after it."""
    out, pool, at = torch.empty(x.shape, dtype=torch.float64, device=DEV), state.clone(), 0
    w, b = w.double(), b.double()
    for l, slot in zip(lens, slots):
        seen = torch.cat([state[slot].double(), x[at:at + l].double()])
        y = b.expand(l, -1).clone()
        for j in range(TAPS):
            y += seen[j:j + l] * w[:, j]
        out[at:at + l] = y * torch.sigmoid(y)
        pool[slot] = seen[l:].to(pool.dtype)
        at += l
    return out, pool


def _exact_scan(s):
    case = s["case"]
    lens, slots = _lens(case), s["slots"].tolist()
    C, P, N = case["channels"], case["headdim"], case["state"]
    xc, pool = _window64(s["x"], s["conv_state"], s["conv_w"], s["conv_b"], lens, slots)
    xc = xc.clamp(-1e3, 1e3)
    dt = torch.nn.functional.softplus(s["dt"].double(), threshold=40.0).clamp(1e-2, 1.0)
    a = torch.exp((dt * s["A"].double().repeat_interleave(P)).clamp(min=NEG_DA))
    u, Bm, Cm = dt * xc, s["B"].double().clamp(-1e3, 1e3), s["C"].double().clamp(-1e3, 1e3)
    state = s["state"].double()
    y = torch.empty(xc.shape, dtype=torch.float64, device=DEV)
    order = sorted(range(len(lens)), key=lambda i: -lens[i])  # the longest first: those still running are a prefix
    starts = s["cu"].tolist()
    first = torch.tensor([starts[i] for i in order], device=DEV)
    which = torch.tensor([slots[i] for i in order], device=DEV)
    h = state[which].reshape(len(lens), C, N)
    for t in range(max(lens)):
        n = sum(1 for i in order if lens[i] > t)
        r = first[:n] + t
        h[:n] = a[r][..., None] * h[:n] + u[r][..., None] * Bm[r][:, None]
        y[r] = torch.einsum("bcn,bn->bc", h[:n], Cm[r])
    state[which] = h.view(len(lens), -1, P, N)
    return {"y": y, "conv_state": pool.double(), "state": state}


def _exact_gdn(s):
    case = s["case"]
    lens, slots = _lens(case), s["slots"].tolist()
    H, D = case["heads"], case["head"]
    done = [_window64(x, s["conv_state"][:, i], w, b, lens, slots)
            for i, (x, w, b) in enumerate(zip(s["x"], s["conv_w"], s["conv_b"]))]
    q, k, v = (t[0].view(-1, H, D) for t in done)
    q, k = (t / torch.sqrt(t.square().sum(-1, keepdim=True) + 1e-12) for t in (q, k))
    b, w, f = (t.double().view(-1, H, D) for t in s["gates"])
    decay = torch.exp(-torch.exp(s["decay_a"].double())[:, None] * torch.nn.functional.softplus(f, threshold=40.0))
    erase, write = torch.sigmoid(b) * k, torch.sigmoid(w) * v.clamp(-50.0, 50.0)
    state = s["state"].double()
    o = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    at = 0
    for l, slot in zip(lens, slots):
        h = state[slot]
        for t in range(at, at + l):
            h = decay[t][..., None] * h
            h = h + torch.einsum("hk,hv->hkv", k[t], write[t] - torch.einsum("hk,hkv->hv", erase[t], h))
            o[t] = torch.einsum("hk,hkv->hv", q[t], h)
        state[slot] = h
        at += l
    return {"y": o.reshape(-1, H * D), "conv_state": torch.stack([t[1] for t in done], 1).double(), "state": state}


def _exact_sample(s):
    logits, noise = s["logits"].double().cpu(), s["noise"].double().cpu()
    B, V = logits.shape
    settings = list(zip(*(s[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p"))))
    tokens, logprobs = [], []
    for l, q, (T, k, p, m) in zip(logits, noise, settings):
        if T == 0:
            T, k = 1.0, 1
        logp = torch.log_softmax(l / T, 0)
        likely, index = torch.sort(logp, descending=True, stable=True)
        prob = likely.exp()
        n = min(k if k > 0 else V, V, max(1, int(((torch.cumsum(prob, 0) - prob) < p).sum())))
        n = min(n, int((prob >= m * prob[0]).sum()), int(torch.isfinite(likely).sum()))
        race = likely[:n] - torch.log(q[index[:n]])
        tokens.append(int(index[:n][race == race.max()].min()))
        logprobs.append(float(logp[tokens[-1]]))
    return {"tokens": torch.tensor(tokens), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "gdn": _exact_gdn, "sample": _exact_sample}[case["op"]](s)
