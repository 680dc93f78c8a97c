"""``training.loss.token_scores`` on the GPU: a given head and a whole bf16 model."""
import pytest
import torch

from atomic_ai_hybrid_b200.config import get_preset
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.training.loss import token_scores
from test_token_scores_cpu import Head, _gradients, _inputs

pytestmark = pytest.mark.gpu
dev = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("T,V,d,chunk", [(2400, 512, 64, 8), (1500, 1001, 40, 256), (1, 128, 64, 2048)])
@pytest.mark.parametrize("store", [False, True])
def test_many_chunks_lose_nothing(T, V, d, chunk, store):
    """As on the CPU: bf16 logits and their gradients, sums in 32 bits; vocabularies and widths with and without kernels."""
    h, w, y = _inputs(T, V, d, BF, dev)
    if T == 1:
        y[:] = 5
    model = Head(h, w)
    if store:
        model.weight._ahb_grad_acc = torch.ones(V, d, device=dev)
    weights = torch.ones(1, T, device=dev), torch.full((1, T), 0.1, device=dev)
    lp, entropy = token_scores(model, {"input_ids": y, "labels": y}, temperature=1.5, chunk=chunk)
    (lp * weights[0] + entropy * weights[1]).sum().backward()
    want = _gradients(h, w, y, 1.5, weights)
    got = model.weight._ahb_grad_acc - 1 if store else model.weight.grad
    assert (model.weight.grad is None) == store
    assert (got.double() - want[3]).norm() <= 1e-2 * want[3].norm(), float((got.double() - want[3]).norm() / want[3].norm())
    assert (model.hidden.grad.double() - want[2]).norm() <= 2e-2 * want[2].norm()
    # a logit of at most 16 is rounded by 2^-8 of itself, and its row's sum by as much
    assert ((lp - want[0]).abs() <= 2 * 16 / 1.5 * 2.0 ** -8 + 1e-4).all()


def test_scores_of_a_model():
    """Log-probabilities and entropies from the same logits' log-softmax in 64 bits, gradients into every parameter."""
    torch.manual_seed(0)
    cfg = get_preset("hybrid_1b", d_model=256, n_heads=2, n_heads_ssm=4, num_layers=2, d_ff=256, n_routed_experts=8, top_k=2,
                     vocab_size=1024, d_state=128, router_noise_std=0.0, dropout_rate=0.0)
    with torch.device(dev):
        model = HybridMoEModel(cfg, compute_dtype=BF)
    ids = torch.randint(0, 1024, (2, 129), device=dev)
    batch = {"input_ids": ids[:, :-1], "labels": ids[:, 1:].clone()}
    batch["labels"][0, :10] = -100
    lp, entropy = token_scores(model, batch, chunk=100)
    with torch.no_grad():
        h, _ = model(batch["input_ids"], return_hidden=True)
        logp = torch.log_softmax((h @ model.lm_weight().to(h.dtype).t()).double(), -1)
    given = batch["labels"] >= 0
    want = logp.gather(2, batch["labels"].clamp(min=0)[..., None])[..., 0] * given
    assert lp.shape == batch["labels"].shape and lp.dtype == F32
    # another run of the layers may route a token near a border elsewhere and sums in another order: most agree, and none by far off
    assert ((lp - want).abs() <= 1e-3 * (1 + want.abs())).double().mean() > 0.9 and ((lp - want).abs() <= 0.2 * (1 + want.abs())).all()
    assert ((entropy + (logp.exp() * logp).sum(-1)).abs() <= 0.1).all()
    (lp.sum() * 0.01 + entropy.sum() * 0.001).backward()
    for n, p in model.named_parameters():
        assert p.grad is None or p.grad.isfinite().all(), n
    assert model.lm_weight().grad is not None and float(model.lm_weight().grad.norm()) > 0
