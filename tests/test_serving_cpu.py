"""Serving on the CPU: the operators' PyTorch forms against direct formulas, a model on kept state against
its forward over whole sequences, generation, refusals."""
import math

import pytest
import torch
import torch.nn.functional as F

from atomic_ai_hybrid_b200 import get_preset, ops
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.ops import reference as R
from atomic_ai_hybrid_b200.serving import DecodeState, Generator, load_weights, serving


def test_selective_scan_is_conv_and_token_serial_scan():
    """From zero state it is the layer's convolution, step and scan (64 bits: differences are rounding)."""
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    B, L, H, P, N = 2, 23, 3, 8, 32
    C = H * P
    x, dt, Bm, Cm, w, b, A = r(B, L, C), r(B, L, C), r(B, L, N), r(B, L, N), r(C, 4), r(C), -r(H).exp()
    conv, state = torch.zeros(B, 3, C, dtype=torch.float64), torch.zeros(B, H, P, N, dtype=torch.float64)
    y = ops.selective_scan(x, dt, A, Bm, Cm, w, b, conv, state)
    xc = R.causal_conv1d(x, w, b, True).view(B, L, H, P)
    step = F.softplus(dt).clamp(1e-2, 1.0).view(B, L, H, P)
    want, s = R.ssd_token_serial(step, A, Bm, Cm, xc)
    torch.testing.assert_close(y.view(want.shape), want, rtol=1e-10, atol=1e-10)
    torch.testing.assert_close(state, s, rtol=1e-10, atol=1e-10)
    assert torch.equal(conv, x[:, -3:])


def test_gdn2_recurrent_is_conv_norm_gates_and_delta_rule():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    B, L, H, D = 2, 9, 2, 16
    d = H * D
    q, k, v, b, w, f = (r(B, L, d) for _ in range(6))
    cw, cb, a = [r(d, 4) for _ in range(3)], [r(d) for _ in range(3)], r(H)
    conv, state = torch.zeros(B, 3, 3, d, dtype=torch.float64), torch.zeros(B, H, D, D, dtype=torch.float64)
    o = ops.gdn2_recurrent(q, k, v, b, w, f, cw, cb, a, conv, state)
    shp = (B, L, H, D)
    qc, kc, vc = (R.causal_conv1d(t, cw[i], cb[i], True).view(shp) for i, t in enumerate((q, k, v)))
    norm = lambda t: t * torch.rsqrt(t.square().sum(-1, keepdim=True) + 1e-12)  # noqa: E731
    gl = -a.exp()[:, None] * F.softplus(f.view(shp))
    want, h = R.gdn2_token_serial(norm(qc), norm(kc), vc.clamp(-50, 50), gl, torch.sigmoid(b).view(shp), torch.sigmoid(w).view(shp))
    torch.testing.assert_close(o.view(shp), want, rtol=1e-10, atol=1e-10)
    torch.testing.assert_close(state, h, rtol=1e-10, atol=1e-10)
    assert torch.equal(conv, torch.stack([q, k, v], 1)[:, :, -3:])


def test_sequences_in_parts_and_padding_slots():
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    T, H, P, N = 12, 2, 4, 32
    C = H * P
    x, dt, Bm, Cm, w, A = r(T, C), r(T, C), r(T, N), r(T, N), r(C, 4), -r(H).exp()
    one = [torch.zeros(4, 3, C, dtype=torch.float64), torch.zeros(4, H, P, N, dtype=torch.float64)]
    two = [t.clone() for t in one]
    cu = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    y = ops.selective_scan(x, dt, A, Bm, Cm, w, None, *one, cu_seqlens=cu(0, 7, 7, 12), slots=cu(2, 0, 1))
    parts = [ops.selective_scan(x[a:e], dt[a:e], A, Bm[a:e], Cm[a:e], w, None, *two, cu_seqlens=cu(0, e - a), slots=cu(s))
             for a, e, s in ((0, 3, 2), (3, 7, 2), (7, 8, 1), (8, 12, 1))]
    torch.testing.assert_close(torch.cat(parts), y)
    for p, q in zip(one, two):
        torch.testing.assert_close(p, q)
    assert (one[1][[0, 3]] == 0).all()
    before = [t.clone() for t in one]
    y = ops.selective_scan(x[:1], dt[:1], A, Bm[:1], Cm[:1], w, None, *one, slots=cu(-1))
    assert (y == 0).all() and all(torch.equal(p, q) for p, q in zip(one, before))
    with pytest.raises(ValueError, match="slot each"):
        ops.selective_scan(x, dt, A, Bm, Cm, w, None, *one)
    with pytest.raises(ValueError, match="cu_seqlens packs"):
        ops.selective_scan(x[None], dt[None], A, Bm[None], Cm[None], w, None, *one, cu_seqlens=cu(0, 12))


def test_sample_rules_and_frequencies():
    logits = torch.tensor([[2.0, 1.0, 2.0, -1.0, float("-inf"), float("nan")]])
    ones = torch.ones(1, 6)
    assert ops.sample(logits, ones, temperature=0.0)[0].item() == 0
    pull = torch.tensor([[9.0, 1.0, 3.0, 1e-6, 1e-9, 1e-9]])
    assert ops.sample(logits, pull)[0].item() == 3
    assert ops.sample(logits, pull, top_k=3)[0].item() == 1
    assert ops.sample(logits, pull, top_k=2)[0].item() == 2
    # masses 1, 1, 0.368, 0.050 of 2.418 by rank: 0.414 are ranked before the second, 0.827 before the third
    assert ops.sample(logits, pull, top_p=0.5)[0].item() == 2
    assert ops.sample(logits, pull, top_p=0.4)[0].item() == 0
    assert ops.sample(logits, pull, top_p=0.3)[0].item() == 0
    assert ops.sample(logits, pull, min_p=0.9)[0].item() == 2
    none = torch.full((1, 3), float("-inf"))
    tok, lp = ops.sample(none, torch.ones(1, 3))
    assert tok.item() == -1 and lp.item() == -math.inf
    p = torch.softmax(torch.tensor([0.3, -0.2, 1.0, 0.0]), 0)
    n = 4000
    noise = torch.empty(n, 4).exponential_(generator=torch.Generator().manual_seed(3))
    count = torch.bincount(ops.sample(p.log()[None].repeat(n, 1), noise)[0], minlength=4).float()
    assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


def _model(preset, **kw):
    torch.manual_seed(0)
    cfg = get_preset(preset, **kw)
    return HybridMoEModel(cfg, compute_dtype=torch.float32).eval(), cfg


@pytest.mark.parametrize("preset,kw", [("tiny", dict(num_layers=2, layer_types=("mamba2", "gdn2"))), ("reference_tiny", {})])
def test_kept_state_equals_whole_sequences(preset, kw):
    """Prompts of uneven lengths, then tokens, give the hidden rows of a forward over the whole sequences.  The two
    run different (fp32) orders of the same sums through a few layers of norms: 1e-3 of the rows' size."""
    model, cfg = _model(preset, **kw)
    L = 64
    ids = torch.randint(0, cfg.vocab_size, (2, L), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        whole, _ = model(ids)
    gen = Generator(model, 4, max_len=L)
    slots, lens = [3, 1], [17, 40]
    logits = gen.prefill([ids[0, :17].tolist(), ids[1, :40].tolist()], slots)
    rows = torch.stack([whole[0, 16], whole[1, 39]])
    want = rows @ model.lm_weight().t()
    assert (logits - want).norm() <= 1e-3 * want.norm()
    for _ in range(20):
        logits = gen.step(torch.stack([ids[i, n] for i, n in enumerate(lens)]), slots)
        want = torch.stack([whole[i, n] for i, n in enumerate(lens)]) @ model.lm_weight().t()
        assert (logits - want).norm() <= 1e-3 * want.norm()
        lens = [n + 1 for n in lens]
    assert gen.state.lengths == [0, 60, 0, 37]


def test_generate_stops_and_repeats():
    model, cfg = _model("tiny", num_layers=2, layer_types=("mamba2", "gdn2"))
    gen = Generator(model, 3)
    prompts = [[1, 2, 3], [7], [5, 6]]
    run = lambda **kw: gen.generate(prompts, 12, top_k=20, generator=torch.Generator().manual_seed(4), **kw)  # noqa: E731
    a, la = run()
    assert [len(t) for t in a] == [12, 12, 12] and all(len(x) == len(y) for x, y in zip(a, la))
    assert run()[0] == a
    greedy = gen.generate(prompts, 6, temperature=0.0)[0]
    assert greedy == gen.generate(prompts, 6, temperature=[0.0, 0.0, 0.0])[0]
    stop = a[1][4]
    b, _ = run(stop_token=stop)
    assert b[1] == a[1][:a[1].index(stop) + 1]
    assert gen.generate(prompts, 0) == ([[], [], []], [[], [], []])


def test_serving_refusals(tmp_path):
    model, cfg = _model("reference_tiny")
    with pytest.raises(ValueError, match="max_len"):
        DecodeState(model, 2)
    gen = Generator(model, 2, max_len=8)
    with pytest.raises(ValueError, match="room for 2"):
        gen.generate([[1]] * 3, 1)
    with pytest.raises(ValueError, match="at least one token"):
        gen.generate([[]], 1)
    with pytest.raises(ValueError, match="max_len=8"):
        gen.prefill([list(range(9))], [0])
    with pytest.raises(ValueError, match="different"):
        gen.prefill([[1], [2]], [0, 0])
    with serving(gen.state, [0], [1]):
        with pytest.raises(RuntimeError, match="not nested"):
            with serving(gen.state, [1], [1]):
                pass
    with pytest.raises(FileNotFoundError):
        load_weights(model, str(tmp_path))


def test_load_weights_from_a_training_checkpoint(tmp_path):
    from atomic_ai_hybrid_b200.ckpt import CheckpointManager
    from atomic_ai_hybrid_b200.training.trainer import Trainer

    model, cfg = _model("tiny", num_layers=2, layer_types=("mamba2", "gdn2"))
    tr = Trainer(model, total_steps=4, compute_dtype=torch.float32, device=torch.device("cpu"))
    mgr = CheckpointManager(str(tmp_path), "latest")
    mgr.save(3, tr, {}, asynchronous=False)
    mgr.finalize()
    torch.manual_seed(9)
    other = HybridMoEModel(cfg, compute_dtype=torch.float32)
    assert load_weights(other, str(tmp_path)) == []
    ids = torch.randint(0, cfg.vocab_size, (1, 64))
    with torch.no_grad():  # the routed experts are stored in bf16
        a, b = model.eval()(ids)[0], other.eval()(ids)[0]
    assert (a - b).norm() <= 2e-2 * a.norm()


def test_expert_parallel_models_are_refused():
    """A rank that holds some of the experts would wait for the others in every layer."""
    from atomic_ai_hybrid_b200.parallel.context import ParallelContext, get_parallel_context, set_parallel_context

    before = get_parallel_context()
    set_parallel_context(ParallelContext(ep_world=2))
    try:
        model, _ = _model("tiny", num_layers=2, layer_types=("mamba2", "gdn2"))
    finally:
        set_parallel_context(before)
    with pytest.raises(ValueError, match="experts"):
        Generator(model, 1)


def test_answering_takes_no_part_in_collectives(monkeypatch):
    """One data-parallel rank may answer while the others do not: nothing of its forward is reduced over them."""
    from atomic_ai_hybrid_b200.models import moe

    model, cfg = _model("tiny", num_layers=2, layer_types=("mamba2", "gdn2"))
    gen = Generator(model, 1)
    want = gen.prefill([[1, 2, 3]], [0])

    def reduced(t):
        raise AssertionError("a collective in a serving call")

    monkeypatch.setattr(moe, "dp_mean", reduced)
    assert torch.equal(gen.prefill([[1, 2, 3]], [0]), want)
    gen.step(torch.tensor([4]), [0])
    with pytest.raises(AssertionError, match="a collective"):
        model(torch.ones(1, 64, dtype=torch.long))


def test_generator_leaves_mode_and_weights_alone():
    """A model in training mode answers without router noise and dropout, and stays in training mode."""
    model, cfg = _model("reference_tiny", dropout_rate=0.5, router_noise_std=1.0)
    want = Generator(model, 1, max_len=16).prefill([[1, 2, 3]], [0])
    model.train()
    before = {n: (p.data_ptr(), p.dtype) for n, p in model.named_parameters()}
    gen = Generator(model, 1, max_len=16)
    assert all(m.training for m in model.modules())
    assert torch.equal(gen.prefill([[1, 2, 3]], [0]), want)
    gen.generate([[1, 2, 3]], 4)
    assert {n: (p.data_ptr(), p.dtype) for n, p in model.named_parameters()} == before


@pytest.mark.parametrize("change", ["load", "step"])
def test_answers_follow_the_weights(change, tmp_path):
    """New weights in the model, Mamba2's decay rates among them, are what the next call of an older Generator runs on."""
    model, cfg = _model("tiny", num_layers=2, layer_types=("mamba2", "gdn2"))
    gen = Generator(model, 1)
    gen.generate([[1, 2, 3]], 3)
    torch.manual_seed(5)
    other = HybridMoEModel(cfg, compute_dtype=torch.float32)
    with torch.no_grad():
        if change == "load":
            model.load_state_dict(other.state_dict())
        else:
            for n, p in model.named_parameters():
                if n.endswith("A_log"):
                    p += 1.0
            other.load_state_dict(model.state_dict())
    ids = [5, 6, 7, 8, 9]
    assert torch.equal(gen.prefill([ids], [0]), Generator(other, 1).prefill([ids], [0]))


def test_other_threads_are_not_serving():
    """While one thread answers, another thread's forward of the same or of another model is an ordinary one, and
    another Generator can answer there."""
    import threading

    model, cfg = _model("tiny", num_layers=2, layer_types=("mamba2", "gdn2"))
    ids = torch.randint(0, cfg.vocab_size, (1, 64), generator=torch.Generator().manual_seed(3))
    with torch.no_grad():
        want = model(ids)[0]
    gen, second = Generator(model, 2), Generator(model, 1)
    answer = second.prefill([[1, 2]], [0])
    got = {}

    def work():
        try:
            with torch.no_grad():
                got["forward"] = model(ids)[0]
                got["other"] = HybridMoEModel(cfg, compute_dtype=torch.float32)(ids)[0]
            got["answer"] = second.prefill([[1, 2]], [0])
        except Exception as e:  # noqa: BLE001
            got["error"] = e

    with serving(gen.state, [0], [64]):
        t = threading.Thread(target=work)
        t.start()
        t.join()
    assert "error" not in got, got["error"]
    assert torch.equal(got["forward"], want) and torch.equal(got["answer"], answer)
    assert all((c[n] == 0).all() for c in gen.state.layers.values() for n in ("conv", "state"))


@pytest.mark.parametrize("prompts,slots,match", [([[1]], [3], "below 3"), ([[1]], [-1], "below 3"), ([[1], [2]], [1, 1], "different"),
                                                 ([[1], []], [0, 1], "at least one"), ([[1]], [0, 1], "at least one"),
                                                 ([[1] * 17], [0], "max_len=16")])
def test_refused_prompts_leave_the_conversations(prompts, slots, match):
    """Slots are checked on the host before anything is reset or indexed (out of range on a GPU they would end the
    process), and a refused call changes nothing."""
    model, cfg = _model("reference_tiny")
    gen = Generator(model, 3, max_len=16)
    gen.prefill([[1, 2, 3], [4, 5]], [0, 1])
    kept = [{n: t.clone() for n, t in c.items()} for c in gen.state.layers.values()]
    with pytest.raises(ValueError, match=match):
        gen.prefill(prompts, slots)
    assert gen.state.lengths == [3, 2, 0]
    assert all(torch.equal(c[n], k[n]) for c, k in zip(gen.state.layers.values(), kept) for n in k)
    if match == "below 3":
        with pytest.raises(ValueError, match=match):
            gen.state.reset(slots)
    assert gen.prefill([[1] * 14], [0], fresh=True).shape == (1, cfg.vocab_size)


def test_forwards_of_other_shapes_are_refused():
    """Inside a call the model takes (1, tokens of the call): other counts would index past the rows, a second batch row
    would be dropped."""
    model, cfg = _model("tiny", num_layers=2, layer_types=("gdn2", "mamba2"))
    state = DecodeState(model, 3)
    for lens, shape in (([5], (1, 4)), ([5], (1, 6)), ([5, 2], (2, 5)), (None, (1, 3)), ([3, 3], (2, 6))):
        with torch.no_grad(), serving(state, list(range(len(lens or [1]))), lens):
            with pytest.raises(ValueError, match="packed"):
                model(torch.ones(shape, dtype=torch.long))
    assert all((c[n] == 0).all() for c in state.layers.values() for n in ("conv", "state"))
    blockdar, _ = _model("reference_tiny", num_layers=3, layer_types=("mla",) * 3)
    with torch.no_grad(), serving(DecodeState(blockdar, 1, 8), [0], [4]):
        with pytest.raises(ValueError, match="packed"):
            blockdar(torch.ones((1, 3), dtype=torch.long))


def test_prompts_outside_the_vocabulary_are_refused():
    """The embedding kernel would take the nearest row for such an id."""
    model, cfg = _model("tiny", num_layers=2, layer_types=("mamba2", "gdn2"))
    gen = Generator(model, 2)
    gen.prefill([[1, 2]], [0])
    for bad in (-1, cfg.vocab_size):
        with pytest.raises(ValueError, match="vocabulary"):
            gen.prefill([[1], [3, bad]], [0, 1])
    assert gen.state.lengths == [2, 0]


def _saved(tmp_path, **kw):
    from atomic_ai_hybrid_b200.ckpt import CheckpointManager
    from atomic_ai_hybrid_b200.training.trainer import Trainer

    model, cfg = _model("tiny", num_layers=2, **kw)
    mgr = CheckpointManager(str(tmp_path), "latest")
    mgr.save(3, Trainer(model, total_steps=4, compute_dtype=torch.float32, device=torch.device("cpu")), {}, asynchronous=False)
    mgr.finalize()


def test_weights_of_another_shape_are_refused(tmp_path):
    """A checkpoint of another model is an error that changes nothing; names that it lacks are returned."""
    _saved(tmp_path, d_ff=256)
    other, cfg = _model("tiny", num_layers=2, d_ff=128)
    before = {n: p.detach().clone() for n, p in other.named_parameters()}
    with pytest.raises(ValueError, match="another shape.*routed_w1"):
        load_weights(other, str(tmp_path))
    assert all(torch.equal(p, before[n]) for n, p in other.named_parameters())
    deeper, _ = _model("tiny", num_layers=3, d_ff=256)
    absent = load_weights(deeper, str(tmp_path))
    assert absent and all(n.startswith("layer_2.") for n in absent)


def test_generate_does_not_answer_with_fresh_weights(tmp_path, capsys):
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "generate.py")
    spec = importlib.util.spec_from_file_location("generate_command", path)
    command = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(command)
    _saved(tmp_path)
    args = ["--preset", "tiny", "--ckpt-root", str(tmp_path), "--prompt", "1,2,3", "--max-new-tokens", "2"]
    command.main(args + ["--layers", "2"])
    assert '"tokens"' in capsys.readouterr().out
    with pytest.raises(SystemExit, match="layer_2"):
        command.main(args + ["--layers", "3"])
    assert capsys.readouterr().out == ""


def test_answers_leave_the_training_diagnostics():
    """What an answer meets is not reported as the training step's, and its forwards take no diagnostic buffer (a
    captured token step would keep that buffer's address)."""
    from atomic_ai_hybrid_b200.utils.diag import DIAG

    for preset, kw in (("tiny", dict(num_layers=2, layer_types=("mamba2", "gdn2"))), ("reference_tiny", {})):
        DIAG.__init__()
        model, cfg = _model(preset, **kw)
        with torch.no_grad():
            for n, p in model.named_parameters():
                if n.endswith("out_proj.kernel"):
                    p[0, 0] = math.nan
        Generator(model, 1, max_len=8).prefill([[1, 2, 3]], [0])
        assert DIAG.buf is None and DIAG.order == []
        with torch.no_grad():
            model(torch.ones(1, 64, dtype=torch.long))
        assert DIAG.order  # an ordinary forward does
