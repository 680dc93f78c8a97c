"""Refusals of the compiled extension reach Python as exceptions, numbers in their text included."""
import pytest
import torch


def test_refusal_with_numbers_is_an_exception():
    ext = pytest.importorskip("atomic_ai_hybrid_b200._ahb_cuda")
    t = torch.zeros(2, 4)
    with pytest.raises(RuntimeError, match="with 8 elements"):
        ext.accumulate_(t, t, 1.0)
