"""Attention layers among recurrent ones on the GPU: prefixes, budgets, captured token steps, scores."""
import json
import os
import subprocess
import sys

import pytest
import torch

from atomic_ai_hybrid_b200.config import get_preset
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.serving import Generator

pytestmark = pytest.mark.gpu
dev = "cuda"


def _model(**kw):
    torch.manual_seed(0)
    cfg = get_preset("reference_tiny", **{**dict(d_model=256, d_ff=256, n_heads=2, n_heads_ssm=4, d_state=64, router_noise_std=0.0,
                                                 dropout_rate=0.0, layer_types=("gdn2", "mla", "mamba2", "mla", "gdn2", "mla")), **kw})
    with torch.device(dev):
        return HybridMoEModel(cfg, compute_dtype=torch.bfloat16).eval(), cfg


def _ids(n, seed, vocab=512):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _close(a, b, tol=5e-2):
    """Logits through six bf16 layers whose sums ran in another order."""
    a, b = a.float(), b.float()
    assert (a - b).norm() <= tol * b.norm(), float((a - b).norm() / b.norm())


@pytest.mark.parametrize("heads", [2, 4])
def test_captured_steps_equal_launched_ones(heads):
    """With a prefix and without, over a budget's cuts, on one generator in turn."""
    torch.manual_seed(0)
    cfg = get_preset("hybrid_1b", d_model=256, n_heads=heads, n_heads_ssm=4, num_layers=4, d_ff=256, n_routed_experts=8, top_k=2,
                     vocab_size=1024, d_state=128, layer_types=("mla", "mamba2", "mla", "mla"))
    with torch.device(dev):
        model = HybridMoEModel(cfg, compute_dtype=torch.bfloat16).eval()
    prompts, P = [_ids(5, 1), _ids(19, 2), _ids(1, 3)], _ids(33, 4)
    gens = [Generator(model, 4, max_len=48, max_positions=200, kv_budget=24, kv_recent=8, cuda_graph=g) for g in (True, False)]
    assert all(g.state.on_device() for g in gens)
    for prefix, seed in ((None, 1), (P, 2), (None, 3), (P, 4)):
        a, b = (g.generate(prompts, 60, top_k=40, prefix=prefix, generator=torch.Generator(device=dev).manual_seed(seed)) for g in gens)
        assert a == b and all(len(t) == 60 for t in a[0])
        assert gens[0].state.rows == gens[1].state.rows and max(gens[0].state.rows) <= 48
        assert gens[0].state.lengths[:3] == [len(p) + 59 + (len(P) if prefix else 0) for p in prompts]
        for g in gens:
            assert g.state.rows_dev.tolist() == g.state.rows and g.state.seen_dev.tolist() == g.state.lengths
    assert len(gens[0]._graphs) == 2 and not gens[1]._graphs


def test_a_failed_capture_leaves_rows_and_masses(monkeypatch):
    from atomic_ai_hybrid_b200 import ops

    model, _ = _model()
    gen = Generator(model, 2, max_len=48, kv_budget=24)
    gen.prefill([[1, 2, 3], [4]], [0, 1])
    kept = [{n: t.clone() for n, t in c.items() if n in ("conv", "state", "mass", "held")} for c in gen.state.layers.values()]

    def broken(*a):
        raise RuntimeError("no sampling today")

    with monkeypatch.context() as m:
        m.setattr(ops, "sample", broken)
        with pytest.raises(RuntimeError, match="no sampling"):
            gen._graph_step([0, 1])
    assert gen.state.lengths == [3, 1] and gen.state.rows == [3, 1] and gen.state.rows_dev.tolist() == [3, 1]
    assert all(torch.equal(c[n], k[n]) for c, k in zip(gen.state.layers.values(), kept) for n in k)


def test_forked_conversations_equal_whole_ones():
    model, _ = _model()
    P, tails = _ids(150, 1), [_ids(4, 2), _ids(37, 3), _ids(1, 4)]
    gen, whole = Generator(model, 4, max_len=200), Generator(model, 3, max_len=400)
    gen.prefill([P], [3])
    gen.fork(3, [0, 1, 2])
    _close(gen.prefill(tails, [0, 1, 2], fresh=False), whole.prefill([P + t for t in tails], [0, 1, 2]))
    for i in range(4):
        t = torch.tensor(_ids(3, 10 + i))
        _close(gen.step(t, [0, 1, 2]), whole.step(t, [0, 1, 2]))


def test_scores():
    """Scores equal the log-softmax of the logits that a prompt's every piece gives."""
    model, _ = _model()
    s, P = _ids(12, 1), _ids(40, 2)
    gen, ref = Generator(model, 2, max_len=64), Generator(model, 1, max_len=64)
    out = gen.score([s], top=4, prefix=P)
    logits = [ref.prefill([P], [0])] + [ref.step(torch.tensor([t]), [0]) for t in s[:-1]]
    logp = torch.log_softmax(torch.cat(logits).double(), -1)
    want = logp.gather(1, torch.tensor(s, device=dev)[:, None])[:, 0]
    got = torch.tensor(out["logprobs"][0], device=dev, dtype=torch.float64)
    assert (got - want).norm() <= 5e-2 * want.norm()
    assert len(out["top_tokens"][0]) == 12 and all(len(t) == 4 for t in out["top_tokens"][0])


def test_generate_command():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    base = [sys.executable, os.path.join(root, "generate.py"), "--preset", "reference_tiny", "--prompt", "1,2,3", "--prompt", "9"]
    run = lambda *a: [json.loads(line) for line in subprocess.run(base + list(a), check=True, capture_output=True, text=True,  # noqa: E731
                                                                 timeout=300).stdout.splitlines() if line.startswith("{")]
    answers = run("--prefix", "4,5,6,7", "--max-new-tokens", "30", "--kv-rows", "20", "--kv-budget", "10")
    assert [len(x["tokens"]) for x in answers] == [30, 30]
    scores = run("--prefix", "4,5,6,7", "--score", "2")
    assert [len(x["logprobs"]) for x in scores] == [3, 1] and all(len(t) == 2 for x in scores for t in x["top_tokens"])
