"""Infinite masses rank above every finite one, and below the newest rows."""
import math

import pytest
import torch

from atomic_ai_hybrid_b200 import ops
from _cache import evict_truth


def evict_case(device):
    top = torch.finfo(torch.float32).max
    mass = torch.tensor([[1.0, top, math.inf, 0.0, top, math.inf, math.nan, -math.inf, 2.0, -top]], device=device)[None].repeat(2, 3, 1)
    M = mass.shape[2]
    g = torch.Generator(device=device).manual_seed(0)
    k, v = (torch.randn(2, 3, M, 8, generator=g, device=device) for _ in range(2))
    held = torch.arange(M, dtype=torch.int32, device=device).expand(2, 3, M).contiguous()
    n = torch.full((2,), M, dtype=torch.int32, device=device)
    return (k, v, mass, held), n, n.clone()


@pytest.mark.parametrize("keep,recent,rows", [(1, 0, [2]), (2, 0, [2, 5]), (3, 0, [5, 1, 2]), (3, 1, [5, 9, 2]), (9, 0, None), (8, 8, None)])
def test_infinite_masses(keep, recent, rows):
    args, n, seen = evict_case("cpu")
    want = evict_truth(*args, n, seen, keep, recent)
    ops.cache_evict(*args, n, seen, keep, recent=recent)
    for a, b in zip(args, want):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    if rows:
        assert args[3][0, 0, :keep].tolist() == rows
