"""rope / qk_norm_rope on overlapping views: the outputs' last dimension is contiguous whatever the input's layout."""

from __future__ import annotations

import pytest
import torch

import helion_b200
from helion_b200 import rope_ops
from oracle import block_oracle
from test_gpu_rope import _check_norm, _close, _rowmax

WIDTH, HEADS = 64, 8


def _sliding(dtype=torch.float32, device="cpu", seed=0):
    """[2, 3, HEADS, WIDTH] windows of one row each: head h begins one element after head h - 1, with a head stride of 1."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, 3, WIDTH + HEADS - 1, generator=g).to(device=device, dtype=dtype).unfold(-1, WIDTH, 1)
    assert x.shape == (2, 3, HEADS, WIDTH) and x.stride()[2:] == (1, 1)
    return x


def test_outputs_of_overlapping_views_on_the_host(monkeypatch):
    """What reaches the C ABI, without a launch."""
    monkeypatch.setattr(rope_ops, "_need_cuda", lambda name, t: None)
    monkeypatch.setattr(rope_ops, "_launch", lambda *a: None)
    monkeypatch.setattr(rope_ops, "_workspace", lambda nbytes, device: torch.empty(8, dtype=torch.uint8))
    monkeypatch.setattr(rope_ops, "_backward_bytes", lambda dim: 8)
    x = _sliding()
    pos, freq = torch.arange(3), torch.ones(WIDTH // 2, dtype=torch.float64)
    w = torch.ones(WIDTH, requires_grad=True)
    outs = [helion_b200.rope(x, pos, freq), *helion_b200.qk_norm_rope(x, x[:, :, :2], w.detach(), w.detach(), pos, freq)]
    q, k = x.detach().requires_grad_(True), x[:, :, 1:].detach().requires_grad_(True)
    made = []
    monkeypatch.setattr(rope_ops, "_row_fields", lambda x, out, *a: made.append(out) or (0,) * 15)
    torch.autograd.grad([t.sum() for t in helion_b200.qk_norm_rope(q, k, w, w, pos, freq)], (q, k))
    assert len(made) == 4  # two outputs, two gradients
    for out in outs + made:
        assert out.stride(-1) == 1 and out.is_contiguous()
    dense = torch.empty(2, HEADS, 3, WIDTH).transpose(1, 2)
    assert rope_ops._heads_like(dense).stride() == dense.stride()  # a dense layout is kept
    assert rope_ops._heads_like(torch.empty(4, 3, 1)).shape == (4, 3, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_overlapping_views(dtype):
    """Against the float64 definitions, within the bounds of every other layout; gradients are taken at the view itself."""
    x, pos = _sliding(dtype, "cuda"), torch.arange(3, device="cuda") + 5
    freq, _ = helion_b200.rope_frequencies(WIDTH)
    every = pos.expand(2, 3)
    _close(helion_b200.rope(x, pos, freq), block_oracle.rope(x, every, freq), dtype, 1.2e-6 * _rowmax(x))
    q, k = x.detach().requires_grad_(True), x[:, :, 2:5].detach().requires_grad_(True)
    assert q.stride(-2) == k.stride(-2) == 1
    dy = torch.randn(2, 3, HEADS, WIDTH, generator=torch.Generator().manual_seed(2)).to("cuda", dtype)
    (dx,) = torch.autograd.grad(helion_b200.rope(q, pos, freq), q, dy)
    _close(dx, block_oracle.rope(dy, every, freq, inverse=True), dtype, 1.2e-6 * _rowmax(dy))
    g = torch.Generator().manual_seed(1)
    weights = [(1 + 0.2 * torch.randn(WIDTH, generator=g)).to("cuda", dtype).requires_grad_(True) for _ in range(2)]
    _check_norm([q, k, *weights], every, freq, dtype, False)
