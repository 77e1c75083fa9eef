"""The slopes of relu in fp32 training belong to the row, not to the batch that it is in. GPU only.

A slope is the sign of z = x W^T + bias. Where z is within its rounding of 0 the order of its sum decides the sign, and an
fp32 z whose sign is saved is one chain of fused multiply-adds over the contraction, then the bias, in every batch."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import helion_b200
from helion_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _chain(x: torch.Tensor, w: torch.Tensor) -> np.ndarray:
    """sum_k x[i, k] w[i, k], k ascending, each step rounded once to 32 bits (the product of two of 24 bits is exact in 64, the
    sum is formed in 64 before its rounding)."""
    x, w = x.numpy().astype(np.longdouble), w.numpy().astype(np.longdouble)
    assert np.finfo(np.longdouble).nmant >= 63
    acc = np.zeros(x.shape[0], dtype=np.float32)
    for k in range(x.shape[1]):
        acc = (x[:, k] * w[:, k] + acc.astype(np.longdouble)).astype(np.float32)
    return acc


@pytest.mark.parametrize(("m", "k", "n"), [(777, 520, 1003), (3, 1024, 300), (64, 517, 130), (1, 2048, 65), (200, 333, 64),
                                           (128, 4096, 128), (2500, 200, 1100)])
def test_slopes_at_an_exact_zero(m, k, n):
    """Each column's bias cancels one row's sum to the last bit: z is 0 there, and relu's slope with it."""
    g = torch.Generator().manual_seed(m + k + n)
    x, w = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g) * k ** -0.5
    row = torch.randint(0, m, (n,), generator=g)
    bias = torch.from_numpy(-_chain(x[row], w))
    dy = torch.zeros(m, n)
    dy[row, torch.arange(n)] = 1.0
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, bias)]
    y = helion_b200.linear(*leaves, activation="relu")
    assert bool((y.detach()[row.to(DEV), torch.arange(n, device=DEV)] == 0).all())
    for grad in torch.autograd.grad(y, leaves, dy.to(DEV)):
        assert bool((grad == 0).all())
    assert _lib.device_status() == 0


def test_a_row_has_the_same_slopes_in_every_batch():
    """The contraction of 777 rows would be split, that of three times as many would not."""
    m, k, n = 777, 520, 1003
    for seed in range(40):
        g = torch.Generator(device=DEV).manual_seed(seed)
        x = torch.randn(m, k, generator=g, device=DEV)
        w = torch.randn(n, k, generator=g, device=DEV) * k ** -0.5
        b, dy = 0.1 * torch.randn(n, generator=g, device=DEV), torch.randn(m, n, generator=g, device=DEV)
        grads = []
        for copies in (1, 3):
            xs = x.repeat(copies, 1).requires_grad_(True)
            y = helion_b200.linear(xs, w, b, activation="relu")
            (dx,) = torch.autograd.grad(y, xs, dy.repeat(copies, 1))
            grads.append(dx[:m])
        # both gradients are sums of the same n products; a slope that differs shifts a row by |dy w|, far beyond
        bound = 2 * n * U * (dy.double().abs() @ w.double().abs())
        assert bool(((grads[0].double() - grads[1].double()).abs() <= bound).all()), seed
