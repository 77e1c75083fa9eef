"""``linear``: a projection with bias, activation and residual in the epilogue of its matrix product.

The projections of a decoder block are ``act(x @ weight.T + bias) + residual`` with some of the three left out. Run as
separate operations, each pass over the product costs a read and a write of it; here they ride on the accumulators of
the GEMM cores that the fused loss uses, and only the result is written (in training also what the activation's
derivative needs). The backward pass forms ``dy * act'`` and the bias gradient in one pass and leaves two products.

``weight`` is ``[out_features, in_features]`` as it is stored, like the LM head's; the reference launches ``matmul``,
``add`` and an activation instead (tritium/ops/matmul.py, add.py, gelu.py, relu.py). A new entry point: ``install()``
rebinds nothing to it.
"""

from __future__ import annotations

from typing import Any

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import FLOAT_DTYPES, _DTYPE_CODE, _differentiated, _launch_scratch, _need_cuda, _need_dtype, _path_flags, _ptr

ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _check(x, weight, bias, activation, residual) -> int:
    _need_cuda("x", x)
    _need_cuda("weight", weight)
    _need_dtype("x", x, FLOAT_DTYPES)
    shape, dtype, device = x.shape, x.dtype, x.device
    if not shape:
        raise ValueError("x must have at least 1 dimension shaped (..., in_features).")
    if weight.dim() != 2:
        raise ValueError("weight must be a 2D tensor shaped (out_features, in_features).")
    n, k = weight.shape
    if shape[-1] != k:
        raise ValueError(f"Shape mismatch: x has last dimension {shape[-1]}, weight expects {k}.")
    if n <= 0 or k <= 0:
        raise ValueError("out_features and in_features must be positive.")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"Shape mismatch: bias has shape {tuple(bias.shape)}, expected ({n},).")
    if residual is not None and residual.shape != (*shape[:-1], n):
        raise ValueError(f"Shape mismatch: residual has shape {tuple(residual.shape)}, expected {(*shape[:-1], n)}.")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is None:
            continue
        if t.dtype != dtype:
            raise ValueError(f"Dtype mismatch: {name} has dtype {t.dtype}, x has dtype {dtype}.")
        if t.device != device:
            raise ValueError(f"Device mismatch: {name} is on {t.device}, x is on {device}.")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of None, 'relu', 'gelu', 'gelu_tanh', 'silu'; got {activation!r}.")
    return act


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t [..., n]`` as rows of contiguous elements and their pitch; copied where its strides allow no such view."""
    n = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, n) if t.numel() else t.new_empty((0, n))
    rows, stride = t.shape[0], t.stride()
    if (stride[1] != 1 and n > 1) or (rows > 1 and stride[0] < n):
        t = t.contiguous()
        return t, n
    return t, stride[0] if rows > 1 else n


def _forward(x, weight, bias, residual, act: int, save: bool):
    """(out [..., N], pre [M, N padded] or None) for x [..., K]."""
    dtype, dev = _DTYPE_CODE[x.dtype], x.device
    x2, ldx = _rows(x)
    w2, ldw = _rows(weight)
    r2, ldr = _rows(residual) if residual is not None else (None, 0)
    m, k = x2.shape
    n = w2.shape[0]
    b = bias.contiguous() if bias is not None else None
    out = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=dev)
    pre = torch.empty((m, (n + 7) // 8 * 8), dtype=x.dtype, device=dev) if save and act else None
    if m == 0:
        return out, pre
    flags = _flags(dtype)
    xp, wp = x2.data_ptr(), w2.data_ptr()
    _launch_scratch("lce_linear_forward",
                    lambda: _lib.lib().lce_linear_forward_workspace_bytes(xp, ldx, wp, ldw, m, n, k, dtype, flags),
                    dev, xp, ldx, wp, ldw, _ptr(b), _ptr(r2), ldr, out.data_ptr(), n, _ptr(pre), m, n, k, act, dtype, flags=flags)
    return out, pre


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _flags(dtype: int) -> int:
    flags = _path_flags()
    return flags & ~_lib.FLAG_FORCE_TC if dtype == _lib.DTYPE_F32 else flags  # fp32 has no tensor-core path


def _backward(dy, x, weight, pre, act: int, need_x: bool, need_w: bool, need_b: bool):
    """(dx, dw, dbias), each or None. Few calls of torch: in autograd's thread each takes several microseconds."""
    dtype, dev = _DTYPE_CODE[x.dtype], x.device
    dy2, ldy = _rows(dy)
    x2, ldx = _rows(x)
    w2, ldw = _rows(weight)
    m, n = dy2.shape
    k = w2.shape[1]
    dx = _empty_like(x) if need_x else None
    dw = _empty_like(weight) if need_w else None
    db = x.new_empty(n) if need_b else None
    flags = _flags(dtype)
    args = (dy2.data_ptr(), ldy, x2.data_ptr(), ldx, w2.data_ptr(), ldw)
    _launch_scratch("lce_linear_backward",
                    lambda: _lib.lib().lce_linear_backward_workspace_bytes(*args, m, n, k, act, dtype, flags),
                    dev, *args, _ptr(pre), _ptr(dx), _ptr(dw), _ptr(db), m, n, k, act, dtype, flags=flags)
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, weight, bias, residual, act):
        out, pre = _forward(x, weight, bias, residual, act, True)
        ctx.save_for_backward(x, weight, pre)
        ctx.act = act
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, *grad_outputs):
        dy = grad_outputs[0]
        x, weight, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            dx, dw, db = _backward(dy, x, weight, pre, ctx.act, need[0], need[1], need[2])
        return dx, dw, db, (dy if need[3] else None), None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` in one pass over the product, rounded once.

    ``x`` is ``[..., in_features]``, ``weight`` ``[out_features, in_features]``, ``bias`` ``[out_features]``,
    ``residual`` shaped like the result; all of one type (bf16, fp16, fp32) and device. ``activation`` is ``None``,
    ``"relu"``, ``"gelu"`` (with the normal distribution function), ``"gelu_tanh"`` or ``"silu"``. Rows may have any
    pitch; inputs whose elements are not contiguous are copied first. fp32 is computed in fp32 throughout. Differentiable
    in ``x``, ``weight``, ``bias`` and ``residual``, not in forward mode; sums are formed in a fixed order. In fp32 relu's
    slopes, which are stored when a gradient is asked for, do not depend on the batch that a row is in."""
    act = _check(x, weight, bias, activation, residual)
    if _differentiated(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, act)
    return _forward(x, weight, bias, residual, act, False)[0]
