"""What capturing a token step does to the conversations, with stand-ins for the CUDA graph (a capture runs the step as written)."""
import contextlib

import pytest
import torch

from atomic_ai_hybrid_b200.config import get_preset
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.serving import DecodeState, Generator


class _Graph:
    def replay(self):
        raise AssertionError("no graph here")


@pytest.fixture
def capturing(monkeypatch):
    """Stand-ins for streams and graphs; a list of whether the step is being captured."""
    now = [False]

    @contextlib.contextmanager
    def graph(*a, **k):
        now[0] = True
        yield
        now[0] = False

    class Stream:
        def __init__(self, *a, **k):
            pass

        def wait_stream(self, other):
            pass

    for name, v in dict(graph=graph, CUDAGraph=_Graph, Stream=Stream, graph_pool_handle=lambda: None, current_stream=Stream,
                        stream=lambda s: contextlib.nullcontext()).items():
        monkeypatch.setattr(torch.cuda, name, v)
    return now


def _ids(n, seed):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _model():
    torch.manual_seed(0)
    return HybridMoEModel(get_preset("reference_tiny", router_noise_std=0.0, dropout_rate=0.0), compute_dtype=torch.float32).eval()


@pytest.mark.parametrize("kw", [dict(max_len=16, kv_budget=8, max_positions=60), dict(max_len=16), dict(max_len=40, max_positions=16)])
@pytest.mark.parametrize("n", [3, 14, 15, 16])
def test_a_capture_needs_no_room_and_leaves_everything(capturing, monkeypatch, kw, n):
    gen = Generator(_model(), 2, **kw)
    st = gen.state
    gen.prefill([_ids(n, 1), _ids(4, 2)], [0, 1])
    kept = [{k: t.clone() for k, t in c.items()} for c in st.layers.values()]
    cuts, cut_back = [], DecodeState.cut_back

    def recorded(self, slots):
        if slots:
            cuts.append((list(slots), capturing[0]))
        cut_back(self, slots)

    monkeypatch.setattr(DecodeState, "cut_back", recorded)
    full = n == 16 and not kw.get("kv_budget")
    with pytest.raises(ValueError, match="would grow past") if full else contextlib.nullcontext():
        gen._graph_step([0, 1])
    assert not cuts  # the replays' loop cuts back, before each one
    assert st.lengths == [n, 4] and st.rows == [n, 4] and st.rows_dev.tolist() == [n, 4] and st.seen_dev.tolist() == [n, 4]
    for c, k in zip(st.layers.values(), kept):
        for name in c:
            for s, rows in enumerate((n, 4)):
                a, b = (t[name][s][:, :rows] if name in ("k", "v", "mass", "held") else t[name][s] for t in (c, k))
                assert torch.equal(a, b), name
