"""``training.loss.token_scores``: the head's weight gradient over many chunks."""
import pytest
import torch

from atomic_ai_hybrid_b200.training.loss import token_scores

BF = torch.bfloat16


class Head(torch.nn.Module):
    """A model whose hidden states are given."""

    def __init__(self, hidden, weight):
        super().__init__()
        self.hidden, self.weight = torch.nn.Parameter(hidden), torch.nn.Parameter(weight)

    def forward(self, ids, return_hidden):
        return self.hidden, []

    def lm_weight(self):
        return self.weight


def _inputs(T, V, d, dtype, device="cpu"):
    g = torch.Generator().manual_seed(0)
    # hidden states around a common one, so that a weight's gradients of all tokens point one way
    h = (torch.randn(1, T, d, generator=g) * 0.25 + torch.randn(d, generator=g)).to(dtype)
    w = (torch.randn(V, d, generator=g) * 0.5).to(dtype)
    y = torch.randint(0, V, (1, T), generator=g)
    y[0, ::7] = -100
    return h.to(device), w.to(device), y.to(device)


def _gradients(h, w, y, temperature, weights):
    """In 64 bits."""
    h, w = (t.detach().double().requires_grad_() for t in (h, w))
    logp = torch.log_softmax(h @ w.t() / temperature, -1)
    lp = torch.where(y >= 0, logp.gather(2, y.clamp(min=0)[..., None])[..., 0], 0.0)
    entropy = -(logp.exp() * logp).sum(-1)
    (lp * weights[0] + entropy * weights[1]).sum().backward()
    return lp, entropy, h.grad, w.grad


@pytest.mark.parametrize("store", [False, True])
def test_many_chunks_lose_nothing(store):
    """600 chunks into a bf16 weight: summed in 32 bits and rounded once.  Logits and their gradients are bf16: each rounded by at most
    2^-8 of its own size in no common direction, a logit's by 2^-8 times its size (at most 8 here) in every probability."""
    T, V, d = 1200, 32, 64
    h, w, y = _inputs(T, V, d, BF)
    model = Head(h, w)
    if store:
        model.weight._ahb_grad_acc = torch.zeros(V, d)
    weights = torch.ones(1, T), torch.full((1, T), 0.1)
    lp, entropy = token_scores(model, {"input_ids": y, "labels": y}, temperature=1.5, chunk=2)
    (lp * weights[0] + entropy * weights[1]).sum().backward()
    want = _gradients(h, w, y, 1.5, weights)
    got = model.weight._ahb_grad_acc if store else model.weight.grad
    if store:
        assert model.weight.grad is None
    assert (got.double() - want[3]).norm() <= 1e-2 * want[3].norm(), float((got.double() - want[3]).norm() / want[3].norm())
    assert (model.hidden.grad.double() - want[2]).norm() <= 2e-2 * want[2].norm()
    assert lp.dtype == torch.float32 and (lp[y == -100] == 0).all()


@pytest.mark.parametrize("chunk", [1, 5, 64])
def test_chunks_do_not_matter(chunk):
    h, w, y = _inputs(17, 23, 8, torch.float32)
    weights = torch.randn(1, 17), torch.randn(1, 17)
    model = Head(h, w)
    lp, entropy = token_scores(model, {"input_ids": y, "labels": y}, temperature=0.7, chunk=chunk)
    (lp * weights[0] + entropy * weights[1]).sum().backward()
    for a, b in zip((lp, entropy, model.hidden.grad, model.weight.grad), _gradients(h, w, y, 0.7, weights)):
        assert torch.allclose(a.double(), b.double(), rtol=1e-4, atol=1e-5)


def test_one_gradient_alone():
    """Scores of which one is used, of a frozen head, and of hidden states without gradient."""
    h, w, y = _inputs(9, 11, 8, torch.float32)
    zero, one = torch.zeros(1, 9), torch.ones(1, 9)
    for i in (0, 1):
        model = Head(h, w)
        token_scores(model, {"input_ids": y, "labels": y}, chunk=4)[i].sum().backward()
        want = _gradients(h, w, y, 1.0, (one, zero) if i == 0 else (zero, one))
        assert torch.allclose(model.weight.grad.double(), want[3], atol=1e-5)
    for frozen in ("hidden", "weight"):
        model = Head(h, w)
        getattr(model, frozen).requires_grad_(False)
        token_scores(model, {"input_ids": y, "labels": y}, chunk=4)[0].sum().backward()
        want = _gradients(h, w, y, 1.0, (one, zero))
        assert getattr(model, frozen).grad is None
        for n, g in (("hidden", want[2]), ("weight", want[3])):
            if n != frozen:
                assert torch.allclose(getattr(model, n).grad.double(), g, atol=1e-5)
    with torch.no_grad():
        assert not token_scores(Head(h, w), {"input_ids": y, "labels": y})[0].requires_grad
