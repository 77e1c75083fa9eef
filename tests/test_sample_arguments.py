"""What sample_logits hands to the C ABI for scalar parameters at the ends of their ranges. No kernel is launched."""

from __future__ import annotations

import pytest
import torch

import helion_b200
from helion_b200 import decode_ops


@pytest.mark.parametrize(("top_k", "given"), [(0, 0), (7, 7), (50, 50), (51, 50), (1 << 40, 50), ((1 << 63) + 3, 50), ((1 << 64) + 1, 50),
                                              (float("inf"), 50)])
def test_a_top_k_of_any_size(monkeypatch, top_k, given):
    """Beyond the vocabulary every top_k is the same: off. The C argument has 64 bits."""
    calls = []
    monkeypatch.setattr(decode_ops, "_need_cuda", lambda name, t: None)
    monkeypatch.setattr(decode_ops, "_launch", lambda what, device, *args: calls.append(args))
    helion_b200.sample_logits(torch.zeros(2, 50), torch.zeros(2), top_k=top_k)
    assert calls[0][10] == given
