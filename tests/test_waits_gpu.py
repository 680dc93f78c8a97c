"""Kernels that give up a wait are heard of where answers are made.  (No wait is made to run out here: the word that they would
leave is put in its place on the host.)"""
import os
import subprocess
import sys

import pytest
import torch

from atomic_ai_hybrid_b200 import ops
from atomic_ai_hybrid_b200.config import get_preset
from atomic_ai_hybrid_b200.models import HybridMoEModel
from atomic_ai_hybrid_b200.ops import kernels as K
from atomic_ai_hybrid_b200.ops._ext import ext
from atomic_ai_hybrid_b200.serving import Generator
from _cache import BF, attention_inputs, check_attention

pytestmark = pytest.mark.gpu
dev = "cuda"


def test_answers_of_a_failed_wait_are_refused(monkeypatch):
    torch.manual_seed(0)
    cfg = get_preset("hybrid_1b", d_model=256, n_heads=2, n_heads_ssm=4, num_layers=2, d_ff=256, n_routed_experts=8, top_k=2,
                     vocab_size=1024, d_state=128, layer_types=("mla", "mamba2"))
    with torch.device(dev):
        gen = Generator(HybridMoEModel(cfg, compute_dtype=BF).eval(), 2, max_len=40)
    ext().gemm_error_reset()
    answers = gen.generate([[1, 2, 3]], 3, temperature=0.0)
    reset = []
    with monkeypatch.context() as m:
        m.setattr(K, "gemm_error", lambda: 66)
        m.setattr(ext(), "gemm_error_reset", lambda: reset.append(1))
        for call in (lambda: gen.generate([[1, 2, 3]], 3), lambda: gen.score([[1, 2, 3]])):
            with pytest.raises(RuntimeError, match="code 66"):
                call()
    assert reset == [1, 1]
    assert gen.generate([[1, 2, 3]], 3, temperature=0.0) == answers and K.gemm_error() == 0


def test_no_wait_of_attention_runs_out():
    ext().gemm_error_reset()
    for lens, had, prefix in (([700, 3], [5, 900], ([400], [0, 0])), ([9, 130], [100, 3], None), ([1] * 12, [5] * 12, ([300], [0] * 12))):
        check_attention(ops.cached_attention, attention_inputs(lens, had, 4, 2, 128, BF, dev, prefix=prefix), 2.0 ** -8)
    assert K.gemm_error() == 0


def test_first_call_in_a_capture():
    """The word is made beside the capture, outside the graph's memory."""
    code = """
import torch
from atomic_ai_hybrid_b200 import ops
from atomic_ai_hybrid_b200.ops import kernels as K
from _cache import BF, attention_inputs, copied
a = attention_inputs([40, 1], [0, 30], 4, 2, 64, BF, "cuda", prefix=([90], [0, 0]))
b, graph = copied(a), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ops.cached_attention(**b)
for _ in range(3):
    graph.replay()
want = y.clone()
del graph, y
torch.cuda.empty_cache()
assert torch.equal(ops.cached_attention(**copied(a)), want) and K.gemm_error() == 0
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([root, os.path.join(root, "tests")]))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
