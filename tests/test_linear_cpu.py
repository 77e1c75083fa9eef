"""linear on the host: refusals, workspace sizes, the C ABI's checks. No kernel is launched here."""

from __future__ import annotations

import pytest
import torch

import helion_b200
from helion_b200 import _lib, linear_ops


@pytest.fixture()
def any_device(monkeypatch):
    monkeypatch.setattr(linear_ops, "_need_cuda", lambda name, t: None)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="x must be a CUDA tensor."):
        helion_b200.linear(torch.randn(4, 8), torch.randn(16, 8))


@pytest.mark.parametrize(("change", "message"), [
    (dict(x=torch.randn(4, 8).double()), "x must have one of these dtypes"),
    (dict(x=torch.tensor(1.0)), "x must have at least 1 dimension"),
    (dict(weight=torch.randn(8)), "weight must be a 2D tensor"),
    (dict(weight=torch.randn(16, 9)), "x has last dimension 8, weight expects 9."),
    (dict(weight=torch.randn(0, 8)), "must be positive"),
    (dict(x=torch.randn(4, 0), weight=torch.randn(16, 0)), "must be positive"),
    (dict(weight=torch.randn(16, 8).half()), "Dtype mismatch: weight has dtype torch.float16"),
    (dict(bias=torch.randn(8)), r"bias has shape \(8,\), expected \(16,\)."),
    (dict(bias=torch.randn(16).half()), "Dtype mismatch: bias"),
    (dict(residual=torch.randn(16)), r"residual has shape \(16,\), expected \(4, 16\)."),
    (dict(residual=torch.randn(4, 16).bfloat16()), "Dtype mismatch: residual"),
    (dict(activation="tanh"), "activation must be one of"),
])
def test_refusals(any_device, change, message):
    args = dict(x=torch.randn(4, 8), weight=torch.randn(16, 8)) | change
    with pytest.raises(ValueError, match=message):
        helion_b200.linear(args["x"], args["weight"], args.get("bias"), activation=args.get("activation"),
                           residual=args.get("residual"))


def test_rows_views_and_copies():
    t = torch.randn(6, 16)
    assert linear_ops._rows(t)[0].data_ptr() == t.data_ptr() and linear_ops._rows(t)[1] == 16
    wide = t[:, 3:9]
    assert linear_ops._rows(wide)[0].data_ptr() == wide.data_ptr() and linear_ops._rows(wide)[1] == 16
    for view in (t.t(), t[:, ::2], torch.randn(16).expand(6, 16), t.view(2, 3, 16).transpose(0, 1)):
        rows, ld = linear_ops._rows(view)
        assert rows.is_contiguous() and ld == view.shape[-1] and torch.equal(rows, view.reshape(-1, view.shape[-1]))
    assert linear_ops._rows(torch.randn(16))[0].shape == (1, 16)
    assert linear_ops._rows(torch.randn(2, 0, 16))[0].shape == (0, 16)


def test_c_abi_checks_and_workspace_sizes():
    L = _lib.lib()
    p = 256  # an aligned address that is never followed: every launching call here is refused

    def forward(x=p, ldx=64, w=p, ldw=64, bias=None, residual=None, ldr=0, out=p, ldo=32, m=4, n=32, k=64, act=0, dtype=0,
                ws=None, ws_bytes=0, flags=0):
        return L.lce_linear_forward(x, ldx, w, ldw, bias, residual, ldr, out, ldo, None, m, n, k, act, dtype, ws, ws_bytes,
                                    flags, None)

    assert forward(n=0) == 1 and forward(k=0, ldx=64) == 1 and forward(m=-1) == 1 and forward(ldx=63) == 1
    assert forward(ldo=31) == 1 and forward(residual=p, ldr=31) == 1 and forward(act=5) == 1 and forward(dtype=3) == 1
    assert forward(x=None) == 1 and forward(w=None) == 1 and forward(out=None) == 1
    assert forward(m=1 << 40) == 6 and forward(dtype=2, flags=_lib.FLAG_FORCE_TC) == 1
    assert forward(m=0) == 0
    # rows off 16-byte boundaries are copied to scratch; it has to be there
    need = L.lce_linear_forward_workspace_bytes(p + 2, 64, p, 64, 4, 32, 64, 0, 0)
    assert need >= 4 * 64 * 2 and forward(x=p + 2, ws=p, ws_bytes=need - 1) == 3 and forward(x=p + 2) == 3
    assert L.lce_linear_forward_workspace_bytes(p, 64, p, 64, 4, 32, 64, 0, 0) == 0
    # a short product is split along its contraction: slabs; a handful of tokens needs none
    assert L.lce_linear_forward_workspace_bytes(p, 8192, p, 8192, 100, 4096, 8192, 0, 0) > 0
    assert L.lce_linear_forward_workspace_bytes(p, 8192, p, 8192, 16, 4096, 8192, 0, 0) == 0

    def backward(dy=p, ldy=32, pre=p, dx=p, dw=p, db=p, m=4, act=2, ws=None, ws_bytes=0):
        return L.lce_linear_backward(dy, ldy, p, 64, p, 64, pre, dx, dw, db, m, 32, 64, act, 0, ws, ws_bytes, 0, None)

    assert backward(dx=None, dw=None, db=None) == 0
    assert backward(pre=None) == 1 and backward(dy=None) == 1 and backward(ldy=31) == 1
    need = L.lce_linear_backward_workspace_bytes(p, 32, p, 64, p, 64, 4, 32, 64, 2, 0, 0)
    assert need >= 4 * 32 * 2 + 32 * 4
