"""A model on kept state on the GPU: prompts, token steps and the graph replay agree with each other and with
the whole-sequence forward."""
import pytest
import torch

from atomic_ai_hybrid_b200 import get_preset, ops
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.serving import Generator, state

pytestmark = pytest.mark.gpu
dev = "cuda"


def _model(**kw):
    torch.manual_seed(0)
    cfg = get_preset("hybrid_1b", **{**dict(d_model=256, n_heads=2, n_heads_ssm=4, num_layers=4, d_ff=256, n_routed_experts=8,
                                            top_k=2, vocab_size=1024, d_state=128, router_noise_std=0.0), **kw})
    with torch.device(dev):
        model = HybridMoEModel(cfg, compute_dtype=torch.bfloat16).eval()
    return model, cfg


def _close(a, b, tol):
    assert torch.isfinite(a).all() and (a.float() - b.float()).norm() <= tol * b.float().norm(), \
        ((a.float() - b.float()).norm() / b.float().norm()).item()


@pytest.mark.parametrize("chunked_from", [64, 768])
def test_kept_state_equals_whole_sequences(chunked_from, monkeypatch):
    """Against the training forward, whose scans multiply bf16 operands (2^-9 each, several in a row: up to 2e-2 a layer)
    where these keep fp32: 5e-2 of the logits' size over two layers.  Every expert is chosen for every token: a
    top-k choice that flips on a near tie is another output altogether."""
    monkeypatch.setattr(state, "GDN_CHUNKED_FROM", chunked_from)
    model, cfg = _model(num_layers=2, n_routed_experts=2, num_experts=3)
    L = 192
    ids = torch.randint(0, cfg.vocab_size, (3, L), generator=torch.Generator().manual_seed(1)).to(dev)
    gen = Generator(model, 5, cuda_graph=False)
    with torch.no_grad():
        whole, _ = model(ids)
        want = whole.float() @ model.lm_weight().float().t()
    slots, lens = [4, 0, 2], [100, 3, 190]
    logits = gen.prefill([ids[i, :n].tolist() for i, n in enumerate(lens)], slots)
    _close(logits, torch.stack([want[i, n - 1] for i, n in enumerate(lens)]), 5e-2)
    for k in range(2):
        logits = gen.step(torch.stack([ids[i, n + k] for i, n in enumerate(lens)]), slots)
        _close(logits, torch.stack([want[i, n + k] for i, n in enumerate(lens)]), 5e-2)
    # a conversation continued by a second prompt (from 64 tokens on: through the chunked scan)
    logits = gen.prefill([ids[0, 102:180].tolist()], [4], fresh=False)
    _close(logits, want[0, 179:180], 5e-2)


def test_graph_replay_equals_single_launches():
    model, cfg = _model()
    prompts = [[5, 6, 7], list(range(70)), [9]]

    def run(graph):
        gen = Generator(model, 4, cuda_graph=graph)
        return gen.generate(prompts, 20, temperature=[0.7, 0.0, 1.2], top_k=40, top_p=0.95,
                            generator=torch.Generator(device=dev).manual_seed(3))

    a, b = run(False), run(True)
    assert a[0] == b[0]
    assert all(len(t) == 20 for t in a[0])


def test_generate_reuses_slots_and_stops():
    model, cfg = _model(num_layers=2)
    gen = Generator(model, 2)
    run = lambda p, **kw: gen.generate(p, 24, top_k=50, generator=torch.Generator(device=dev).manual_seed(5), **kw)[0]  # noqa: E731
    first = run([[1, 2], [3]])
    assert run([[1, 2], [3]]) == first
    stop = first[0][10]
    assert run([[1, 2], [3]], stop_token=stop)[0] == first[0][:first[0].index(stop) + 1]


def test_blockdar_with_mla():
    """The reference's layout (head dim 64, MLA layers, PyTorch attention over kept keys) runs and repeats itself
    whether its prompt comes at once or in two pieces."""
    torch.manual_seed(0)
    cfg = get_preset("reference_tiny", router_noise_std=0.0, dropout_rate=0.0)
    with torch.device(dev):
        model = HybridMoEModel(cfg, compute_dtype=torch.bfloat16).eval()
    ids = torch.randint(0, cfg.vocab_size, (50,), generator=torch.Generator().manual_seed(2)).tolist()
    gen = Generator(model, 2, max_len=64)
    a = gen.prefill([ids], [0])
    gen.prefill([ids[:30]], [1])
    b = gen.prefill([ids[30:]], [1], fresh=False)
    _close(b, a, 5e-2)
    assert len(gen.generate([ids[:5], ids[:9]], 4, temperature=0.0)[0][1]) == 4
    assert ops.get_impl() == "cuda"
