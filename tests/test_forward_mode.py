"""Forward-mode derivatives: no operator has them, so each refuses an input that carries a tangent instead of dropping it.
The refusal comes from the operators' autograd functions; what they launch is replaced here, so that no device is needed."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import helion_b200
from helion_b200 import ce_ops, linear_ops, matmul_ops, norm_ops, ops, rope_ops

M, K, N = 4, 16, 8
LABELS = torch.zeros(M, dtype=torch.int64)
POSITIONS, FREQUENCIES = torch.zeros(M, dtype=torch.int64), torch.ones(K // 2, dtype=torch.float64)


def _heads(x):
    return x.unflatten(-1, (1, K))


# name -> (shapes of the differentiable inputs, the call)
CALLS = {
    "linear": ([(M, K), (N, K), (N,), (M, N)], lambda x, w, b, r: helion_b200.linear(x, w, b, activation="gelu", residual=r)),
    "rope": ([(M, K)], lambda x: helion_b200.rope(_heads(x), POSITIONS, FREQUENCIES)),
    "qk_norm_rope": ([(M, K), (M, K), (K,), (K,)],
                     lambda q, k, wq, wk: helion_b200.qk_norm_rope(_heads(q), _heads(k), wq, wk, POSITIONS, FREQUENCIES)[0]),
    "matmul": ([(M, K), (K, N)], helion_b200.matmul),
    "rmsnorm": ([(M, K), (K,)], helion_b200.rmsnorm),
    "residual_rmsnorm": ([(M, K), (M, K), (K,)], lambda *a: helion_b200.residual_rmsnorm(*a)[0]),
    "cross_entropy": ([(M, N)], lambda x: helion_b200.cross_entropy(x, LABELS)),
    "linear_cross_entropy": ([(M, K), (N, K)], lambda x, w: helion_b200.linear_cross_entropy(x, w, LABELS)),
}


@pytest.fixture(autouse=True)
def _no_launches(monkeypatch):
    for module in (ce_ops, linear_ops, matmul_ops, norm_ops, ops, rope_ops):
        monkeypatch.setattr(module, "_need_cuda", lambda name, t: None)
    monkeypatch.setattr(linear_ops, "_forward", lambda x, w, *a: (torch.zeros(M, N), None))
    monkeypatch.setattr(rope_ops, "_rope", lambda x, *a: torch.zeros(x.shape))
    monkeypatch.setattr(rope_ops, "_qk_forward", lambda q, k, *a: (torch.zeros(q.shape), torch.zeros(k.shape)))
    monkeypatch.setattr(matmul_ops, "_product", lambda a, b: torch.zeros(M, N))
    monkeypatch.setattr(norm_ops, "_forward", lambda x, *a: (torch.zeros(M, K), torch.zeros(M, K), torch.zeros(M)))
    for module in (ce_ops, ops):
        monkeypatch.setattr(module, "_forward", lambda *a: (torch.zeros(()), torch.zeros(M)))


@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_is_refused(name):
    shapes, call = CALLS[name]
    inputs = [torch.randn(s) for s in shapes]
    call(*inputs)
    with forward_ad.dual_level():
        call(*inputs)  # an open level alone refuses nothing
        for i in range(len(inputs)):
            some = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(inputs)]
            with pytest.raises(RuntimeError):
                call(*some)
            with torch.no_grad(), pytest.raises(RuntimeError):
                call(*some)
    for i in range(len(inputs)):
        def one(t, i=i):
            return call(*(t if j == i else u for j, u in enumerate(inputs)))
        with pytest.raises(RuntimeError):
            torch.func.jvp(one, (inputs[i],), (torch.ones_like(inputs[i]),))
    torch.func.jvp(lambda t: 2 * t + call(*inputs).sum(), (torch.ones(3),), (torch.ones(3),))  # none of its inputs has one
    call(*(t.requires_grad_(True) for t in inputs))
