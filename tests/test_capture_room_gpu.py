"""Answers whose token step is captured while one row, or none, is left."""
import pytest
import torch

from atomic_ai_hybrid_b200.config import get_preset
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.serving import Generator

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.fixture(scope="module")
def model():
    torch.manual_seed(0)
    cfg = get_preset("hybrid_1b", d_model=256, n_heads=2, n_heads_ssm=4, num_layers=4, d_ff=256, n_routed_experts=8, top_k=2,
                     vocab_size=1024, d_state=128, layer_types=("mla", "mamba2", "mla", "mla"))
    with torch.device(dev):
        return HybridMoEModel(cfg, compute_dtype=torch.bfloat16).eval()


@pytest.mark.parametrize("n,new,kw", [(47, 30, dict(max_len=48, max_positions=90, kv_budget=24)), (48, 30, dict(max_len=48, max_positions=90, kv_budget=24)),
                                      (47, 2, dict(max_len=48)), (47, 2, dict(max_len=80, max_positions=48))])
def test_captured_answers_equal_launched_ones(model, n, new, kw):
    ids = lambda n, s: torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(s)).tolist()  # noqa: E731
    gens = [Generator(model, 2, cuda_graph=g, **kw) for g in (True, False)]
    a, b = (g.generate([ids(n, 1), ids(5, 2)], new, top_k=40, generator=torch.Generator(device=dev).manual_seed(3)) for g in gens)
    assert a == b and [len(t) for t in a[0]] == [new, new]
    assert len(gens[0]._graphs) == 1
    for g in gens:
        assert g.state.lengths == [n + new - 1, 5 + new - 1] and g.state.rows_dev.tolist() == g.state.rows
        assert g.state.seen_dev.tolist() == g.state.lengths
    for x, y in zip(*(g.state.layers.values() for g in gens)):
        if "mass" in x:
            for s, rows in enumerate(gens[0].state.rows):
                assert torch.equal(x["held"][s, :, :rows], y["held"][s, :, :rows])
                assert torch.equal(x["mass"][s, :, :rows], y["mass"][s, :, :rows])
