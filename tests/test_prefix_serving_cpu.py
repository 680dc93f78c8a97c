"""Conversations that share a prefix, that are cut back to a budget, and scores of sequences, through a whole model."""
import pytest
import torch

from atomic_ai_hybrid_b200.config import get_preset
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.serving import DecodeState, Generator, serving


def _model(preset="reference_tiny", **kw):
    torch.manual_seed(0)
    cfg = get_preset(preset, **{"router_noise_std": 0.0, "dropout_rate": 0.0, **kw})
    return HybridMoEModel(cfg, compute_dtype=torch.float32).eval(), cfg


def _ids(n, seed, vocab=512):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _close(a, b, tol=1e-3):
    """Two fp32 orders of the same sums through a few layers of norms."""
    assert (a - b).norm() <= tol * b.norm(), float((a - b).norm() / b.norm())


@pytest.mark.parametrize("preset,kw", [("reference_tiny", {}), ("tiny", dict(num_layers=2, layer_types=("mamba2", "gdn2")))])
def test_forked_conversations_equal_whole_ones(preset, kw):
    model, cfg = _model(preset, **kw)
    P, tails = _ids(23, 1), [_ids(4, 2), _ids(9, 3), _ids(1, 4)]
    gen, whole = Generator(model, 5, max_len=40), Generator(model, 3, max_len=80)
    gen.prefill([P], [4])
    gen.fork(4, [2, 0, 1])
    assert gen.state.lengths == [23, 23, 23, 0, 23]
    a = gen.prefill(tails, [2, 0, 1], fresh=False)
    b = whole.prefill([P + t for t in tails], [0, 1, 2])
    _close(a, b)
    for i in range(6):
        t = torch.tensor(_ids(3, 10 + i))
        _close(gen.step(t, [2, 0, 1]), whole.step(t, [0, 1, 2]))
    assert gen.state.lengths == [23 + 9 + 6, 23 + 1 + 6, 23 + 4 + 6, 0, 23]
    # conversations with and without a prefix in one call
    gen.prefill([_ids(5, 30)], [3])
    whole2 = Generator(model, 1, max_len=80)
    whole2.prefill([_ids(5, 30)], [0])
    t = torch.tensor([7, 8])
    both = gen.step(t, [0, 3])
    _close(both[1:], whole2.step(t[1:], [0]))


def test_fork_refuses_and_protects():
    model, _ = _model()
    gen = Generator(model, 4, max_len=30)
    gen.prefill([_ids(10, 1), _ids(3, 2)], [0, 3])
    gen.fork(0, [1, 2])
    with pytest.raises(ValueError, match="slot 0 is shared"):
        gen.step(torch.tensor([1]), [0])
    with pytest.raises(ValueError, match="slot 0 is shared"):
        gen.prefill([[1]], [0])
    with pytest.raises(ValueError, match="slot 0 is shared"):
        gen.fork(3, [0])
    with pytest.raises(ValueError, match="forked from slot 0"):
        gen.fork(1, [3])
    with pytest.raises(ValueError, match="into itself"):
        gen.fork(3, [1, 3])
    with pytest.raises(ValueError, match="slots must be different"):
        gen.fork(7, [1])
    assert gen.state.lengths == [10, 10, 10, 3] and gen.state.prefix == [-1, 0, 0, -1]
    gen.fork(3, [1, 2])  # the forks are new conversations: slot 0 is free again
    gen.step(torch.tensor([1]), [0])
    gen.prefill([[1], [2], [3], [4]], [0, 1, 2, 3])  # all at once, the shared one among them
    assert gen.state.prefix == [-1] * 4 and gen.state.lengths == [1] * 4
    with pytest.raises(ValueError, match="max_positions=60"):
        gen.prefill([_ids(30, 1)], [3])
        gen.fork(3, [0])
        gen.prefill([_ids(31, 1)], [0], fresh=False)


def test_generate_with_a_prefix():
    model, _ = _model()
    P, prompts = _ids(17, 1), [_ids(3, 2), _ids(6, 3)]
    run = lambda **kw: Generator(model, 3, max_len=60).generate(  # noqa: E731
        **kw, max_new_tokens=10, temperature=[0.0, 0.9], top_k=20, generator=torch.Generator().manual_seed(3))
    a, b = run(prompts=prompts, prefix=P), run(prompts=[P + p for p in prompts])
    assert a[0] == b[0]
    for x, y in zip(a[1], b[1]):
        assert all(abs(p - q) <= 1e-3 * (1 + abs(q)) for p, q in zip(x, y))
    gen = Generator(model, 3, max_len=60)
    for _ in range(2):  # prefixes and none in turn, on the same slots
        assert gen.generate(prompts, 5, temperature=0.0, prefix=P)[0] == gen.generate([P + p for p in prompts], 5, temperature=0.0)[0]
        gen.generate(prompts + [[5]], 2)
    with pytest.raises(ValueError, match="3 prompts, room for 2"):
        gen.generate(prompts + [[5]], 2, prefix=P)
    with pytest.raises(ValueError, match="at least one token"):
        gen.generate(prompts, 2, prefix=[])


def test_scores_equal_whole_sequences():
    model, cfg = _model()
    seqs, P = [_ids(30, 1), _ids(64, 2)[:64], _ids(1, 3)], _ids(20, 4)
    gen = Generator(model, 4, max_len=100)

    def want(ids):
        pad = -len(ids) % 64
        with torch.no_grad():
            h, _ = model(torch.tensor([ids + [0] * pad]))
        return torch.log_softmax((h[0, :len(ids)] @ model.lm_weight().detach().t()).double(), -1)

    def held(out, i, logp, tokens):
        assert len(out["logprobs"][i]) == len(tokens)
        for t, y in enumerate(tokens):
            p = logp[t]
            assert abs(out["logprobs"][i][t] - float(p[y])) <= 2e-3 * (1 + abs(float(p[y])))
            assert abs(out["entropy"][i][t] + float((p.exp() * p).sum())) <= 2e-3 * 10
            best = torch.tensor(out["top_logprobs"][i][t])
            assert (best[:-1] >= best[1:]).all() and len(out["top_tokens"][i][t]) == 3
            assert (best - p[out["top_tokens"][i][t]]).abs().max() <= 2e-2

    out = gen.score(seqs, top=3)
    for i, s in enumerate(seqs):
        held(out, i, want(s), s[1:])
    out = gen.score(seqs, top=3, prefix=P)
    for i, s in enumerate(seqs):
        held(out, i, want(P + s)[len(P) - 1:], s)
    assert set(gen.score(seqs)) == {"logprobs", "entropy"}
    assert gen.score([[4]], top=2) == {"logprobs": [[]], "entropy": [[]], "top_tokens": [[]], "top_logprobs": [[]]}


def test_score_in_pieces(monkeypatch):
    from atomic_ai_hybrid_b200.serving import generate
    model, cfg = _model()
    seqs = [_ids(30, 1), _ids(7, 2)]
    a = Generator(model, 2, max_len=40).score(seqs, top=2)
    monkeypatch.setattr(generate, "SCORE_LOGITS", 4 * cfg.vocab_size)
    b = Generator(model, 2, max_len=40).score(seqs, top=2)
    assert a["top_tokens"] == b["top_tokens"]
    assert torch.allclose(torch.tensor(a["logprobs"][0]), torch.tensor(b["logprobs"][0]), rtol=1e-5, atol=1e-5)


def test_conversations_go_on_within_a_budget():
    """While nothing is cut the answers are those without a budget; afterwards rows stay bounded and the newest are held."""
    model, _ = _model()
    free = Generator(model, 2, max_len=200)
    gen = Generator(model, 2, max_len=24, max_positions=100, kv_budget=12, kv_recent=6)
    prompts = [_ids(10, 1), _ids(14, 2)]
    a, b = gen.prefill(prompts, [0, 1]), free.prefill(prompts, [0, 1])
    _close(a, b)
    for i in range(60):
        t = torch.tensor(_ids(2, 50 + i))
        a, b = gen.step(t, [0, 1]), free.step(t, [0, 1])
        if i < 10:
            _close(a, b)
        assert a.isfinite().all() and max(gen.state.rows) <= 24
    assert gen.state.lengths == [70, 74]
    for c in gen.state.layers.values():
        if "held" in c:
            for s in (0, 1):
                n = gen.state.rows[s]
                for row in c["held"][s, :, :n].tolist():
                    assert len(set(row)) == n and set(range(gen.state.lengths[s] - 6, gen.state.lengths[s])) <= set(row)
                # weights of a token sum to one, and no row is older than it was when it came
                assert (c["mass"][s, :, :n] >= 0).all()
    assert gen.state.rows_dev.tolist() == gen.state.rows and gen.state.seen_dev.tolist() == gen.state.lengths
    with pytest.raises(ValueError, match="max_len=24"):
        gen.prefill([_ids(13, 1)], [0], fresh=False)  # more than the budget leaves room for
    with pytest.raises(ValueError, match="max_positions=100"):
        gen.state.lengths[0] = 95
        gen.prefill([_ids(7, 1)], [0], fresh=False)


def test_evicted_rows_are_those_with_least_mass():
    """A budget of all but one row gives up the row that got least, in every layer and head, and leaves its weight to the others."""
    model, _ = _model()
    st = DecodeState(model, 1, max_len=12, max_positions=40, budget=11, recent=2)
    gen = Generator(model, 1, max_len=12)
    gen.state = st
    gen.prefill([_ids(12, 1)], [0])
    before = {m: {n: t.clone() for n, t in c.items()} for m, c in st.layers.items() if "mass" in c}
    assert all(abs(float(c["mass"][0].sum(-1).mean()) - 12) <= 1e-4 for c in before.values())  # 12 tokens, each a weight of one
    st.cut_back([0])
    for m, c in before.items():
        for h in range(c["mass"].shape[1]):
            worst = int(c["mass"][0, h, :10].argmin())
            assert worst not in st.layers[m]["held"][0, h, :11].tolist()
    assert st.rows == [11] and st.lengths == [12]


def test_budget_refuses():
    model, _ = _model()
    for kw in (dict(kv_budget=8), dict(kv_budget=9), dict(kv_budget=4, kv_recent=5), dict(kv_budget=4, kv_recent=-1)):
        with pytest.raises(ValueError, match="budget must be below max_len=8"):
            Generator(model, 1, max_len=8, **kw)
    gen = Generator(model, 2, max_len=8, max_positions=20)
    with pytest.raises(ValueError, match="needs a budget"):
        gen.state.cut_back([0])
    gen = Generator(model, 2, max_len=8, max_positions=20, kv_budget=4)
    gen.prefill([_ids(6, 1)], [0])
    gen.fork(0, [1])
    with pytest.raises(ValueError, match="slot 0 is shared"):
        gen.state.cut_back([0])


def test_an_error_in_a_forward_leaves_the_rows():
    model, _ = _model()
    gen = Generator(model, 2, max_len=20)
    gen.prefill([[1, 2, 3]], [0])
    with pytest.raises(RuntimeError, match="on the way"):
        with serving(gen.state, [0]):
            raise RuntimeError("on the way")
    assert gen.state.rows == [3, 0] and gen.state.rows_dev.tolist() == [3, 0] and gen.state.lengths == [3, 0]

