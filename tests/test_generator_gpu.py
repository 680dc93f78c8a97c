"""What a Generator leaves of the model that it is given, and what it sees of that model's changes, on the GPU."""
import pytest
import torch

from atomic_ai_hybrid_b200 import get_preset, ops
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.serving import DecodeState, Generator, compute_weights, serving

pytestmark = pytest.mark.gpu
dev = "cuda"


def _model(**kw):
    torch.manual_seed(0)
    cfg = get_preset("hybrid_1b", **{**dict(d_model=256, n_heads=2, n_heads_ssm=4, num_layers=4, d_ff=256, n_routed_experts=8,
                                            top_k=2, vocab_size=1024, d_state=128), **kw})
    with torch.device(dev):
        return HybridMoEModel(cfg, compute_dtype=torch.bfloat16), cfg


def _weights(model):
    return {n: (p.data_ptr(), p.dtype, p.detach().clone()) for n, p in model.named_parameters()}


def _unchanged(model, before):
    for n, p in model.named_parameters():
        ptr, dtype, value = before[n]
        assert p.data_ptr() == ptr and p.dtype is dtype and torch.equal(p, value), n


def _direct(model, ids):
    """Logits after ``ids`` on a state of their own, without a Generator."""
    with torch.no_grad(), serving(DecodeState(model, 1), [0], [len(ids)]):
        h, _ = model(torch.tensor([ids], device=dev))
    return h[0, -1:] @ model.lm_weight().to(h.dtype).t()


@pytest.mark.parametrize("training", [True, False])
def test_generator_leaves_the_model_alone(training):
    """Weights, their dtypes (the router's fp32 among them) and the mode; its logits are those of the model as it was
    before, from the same kernels on the same weights: equal up to the order of sums that atomics may take."""
    model, cfg = _model()
    model.train(training)
    before = _weights(model)
    ids = torch.randint(0, cfg.vocab_size, (40,), generator=torch.Generator().manual_seed(1)).tolist()
    want = _direct(model, ids)
    gen = Generator(model, 2)
    got = gen.prefill([ids], [1])
    assert (got - want).float().norm() <= 1e-3 * want.float().norm()
    gen.generate([ids, [3]], 6)
    _unchanged(model, before)
    assert all(m.training == training for m in model.modules())


def test_generating_between_training_steps():
    """A trainer's model answers and goes on training: its parameters stay the store's views."""
    from atomic_ai_hybrid_b200.training.trainer import Trainer

    model, cfg = _model(num_layers=2)
    tr = Trainer(model, total_steps=8, optimizer="adamw", device=torch.device(dev))
    g = torch.Generator().manual_seed(2)
    first = _weights(model)
    for _ in range(3):
        ids = torch.randint(0, 16, (2, 65), generator=g).to(dev)
        loss = tr.train_step([{"input_ids": ids[:, :-1], "labels": ids[:, 1:]}])["loss"]
        assert torch.isfinite(loss)
        before = _weights(model)
        compute_weights(model)
        tokens, _ = Generator(model, 2).generate([[1, 2, 3], [4]], 5, top_k=8)
        assert [len(t) for t in tokens] == [5, 5]
        _unchanged(model, before)
        for s in tr.store.segs:
            assert s.param.data_ptr() == tr.store.compute_view(s).data_ptr(), s.name
    assert not torch.equal(model.layer_0.moe.router, first["layer_0.moe.router"][2])  # the steps reached the model
    tr.close()


def test_compute_weights_keeps_what_training_keeps():
    """Matrices in bf16, the router and the vectors in fp32; the logits are the same, as every product rounds its
    matrix to bf16 either way."""
    model, cfg = _model(num_layers=2)
    want = _direct(model, [5, 6, 7])
    assert compute_weights(model) is model
    for n, p in model.named_parameters():
        assert p.dtype is (torch.float32 if p.ndim < 2 or n.endswith("router") else torch.bfloat16), n
    got = _direct(model, [5, 6, 7])
    # the convolutions' taps (2^-9 of their values) are the one difference, seen through two layers
    assert (got - want).float().norm() <= 2e-2 * want.float().norm()


def test_captured_steps_follow_the_weights():
    """Weights changed in place after a graph was captured, Mamba2's decay rates among them, are those it runs on."""
    model, cfg = _model(num_layers=2)
    gen = Generator(model, 2)
    run = lambda g: g.generate([[1, 2, 3], [9]], 24, top_k=50, generator=torch.Generator(device=dev).manual_seed(4))  # noqa: E731
    old = run(gen)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith("A_log") or n.endswith("final_norm.scale"):
                p += 0.5
    new = run(gen)
    assert new[0] == run(Generator(model, 2))[0] and new[1] != old[1]


@pytest.mark.parametrize("kw", [dict(d_model=128, d_ff=128), dict(d_state=16), dict(n_heads=8), dict(compute_dtype=torch.float32), dict()])
@pytest.mark.parametrize("impl", ["cuda", "eager"])
def test_sizes_without_kernels_are_launched(kw, impl):
    """A layer that reads on the host cannot be captured: the token step is launched, with the same answer as ever."""
    kw = dict(kw)
    dtype = kw.pop("compute_dtype", torch.bfloat16)
    model, cfg = _model(num_layers=2, **kw)
    model.compute_dtype = dtype
    run = lambda graph: Generator(model, 2, cuda_graph=graph).generate(  # noqa: E731
        [[1, 2, 3], [9]], 6, top_k=50, generator=torch.Generator(device=dev).manual_seed(4))
    with ops.impl(impl):
        gen = Generator(model, 2)
        assert gen.state.on_device() == (not kw and dtype is torch.bfloat16 and impl == "cuda")
        assert run(True)[0] == run(False)[0]


@pytest.mark.parametrize("move", ["compute_weights", "trainer"])
def test_captured_steps_find_moved_weights(move):
    """Parameters that moved to other memory after a capture (into a trainer's store, to another dtype) and changed
    there: the graph is captured again."""
    from atomic_ai_hybrid_b200.training.trainer import Trainer

    model, cfg = _model(num_layers=2)
    gen = Generator(model, 2)
    run = lambda g: g.generate([[1, 2, 3], [9]], 24, top_k=50, generator=torch.Generator(device=dev).manual_seed(4))  # noqa: E731
    old = run(gen)
    if move == "compute_weights":
        compute_weights(model)
    else:
        tr = Trainer(model, total_steps=4, optimizer="adamw", device=torch.device(dev))
    with torch.no_grad():
        for n, p in model.named_parameters():
            if p.ndim == 2 and not n.startswith("embed"):
                p *= 0.5
    new = run(gen)
    assert new[0] == run(Generator(model, 2))[0] and new[1] != old[1]
    if move == "trainer":
        tr.close()


def test_a_failed_capture_leaves_the_conversations(monkeypatch):
    """States and lengths after a step that cannot be captured are those before it."""
    model, cfg = _model(num_layers=2)
    gen = Generator(model, 2)
    gen.prefill([[1, 2, 3], [4]], [0, 1])
    kept = [{n: t.clone() for n, t in c.items()} for c in gen.state.layers.values()]

    def broken(*a):
        raise RuntimeError("no sampling today")

    with monkeypatch.context() as m:
        m.setattr(ops, "sample", broken)
        with pytest.raises(RuntimeError, match="no sampling"):
            gen._graph_step([0, 1])
    assert gen.state.lengths == [3, 1] and not gen._graphs
    assert all(torch.equal(c[n], k[n]) for c, k in zip(gen.state.layers.values(), kept) for n in k)
    assert [len(t) for t in gen.generate([[1, 2, 3], [4]], 4)[0]] == [4, 4]


def test_graphs_of_many_batch_sizes_are_bounded():
    """Answers to every batch size, twice around: a bounded number of graphs is kept, their buffers are shared, and
    memory does not grow."""
    from atomic_ai_hybrid_b200.serving import generate

    model, cfg = _model(num_layers=2, vocab_size=50304)
    gen, plain = Generator(model, 12), Generator(model, 12, cuda_graph=False)
    held = []
    for turn in range(3):
        for B in range(1, 13):
            run = lambda g: g.generate([[i + 1, 7] for i in range(B)], 4, top_k=50,  # noqa: E731
                                       generator=torch.Generator(device=dev).manual_seed(B))
            got = run(gen)
            assert len(gen._graphs) <= generate.MAX_GRAPHS
            assert turn or got[0] == run(plain)[0]
        torch.cuda.synchronize()
        held.append(torch.cuda.memory_reserved())
    assert held[2] <= held[1]


def test_captures_on_the_models_device(monkeypatch):
    """The capture runs on a stream of the model's device, whichever device is the current one (without a stream
    PyTorch takes one of the device that was current at the process's first capture: kernels elsewhere are not
    captured)."""
    streams, graph = [], torch.cuda.graph

    def capture(*a, **kw):
        streams.append(kw.get("stream"))
        return graph(*a, **kw)

    monkeypatch.setattr(torch.cuda, "graph", capture)
    home = torch.device(dev, torch.cuda.device_count() - 1)
    model, cfg = _model(num_layers=2)
    gen = Generator(model.to(home), 2)
    with torch.cuda.device(0):
        tokens = gen.generate([[1, 2, 3], [9]], 6, temperature=0.0)[0]
    assert len(streams) == 1 and streams[0].device == home
    assert tokens == Generator(model, 2, cuda_graph=False).generate([[1, 2, 3], [9]], 6, temperature=0.0)[0]
