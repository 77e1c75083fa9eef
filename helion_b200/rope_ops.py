"""Rotary positions, alone (``rope``) and behind the RMS norm of every query and key head (``qk_norm_rope``).

They stand between ``rmsnorm`` and attention in a decoder block: the projection's heads are normalised, rotated by
their positions and handed on, in one pass over the data. Heads are ``[batch, seq, heads, dim]`` or
``[tokens, heads, dim]`` tensors of any strides with a contiguous last dimension - slices of a fused query/key/value
projection and ``transpose(1, 2)`` views of a ``[batch, heads, seq, dim]`` layout are taken as they are; a single
token per sequence is ``seq = 1``.

The angles are ``positions * frequencies``, formed in 64 bits, so any position is as exact as the first ones and
nothing is tabulated per length. ``rope_frequencies`` makes the frequencies, scaled for long contexts where asked.
The reference has a rotary op of its own (tritium/ops/rope.py); these are new entry points and ``install()`` rebinds
nothing to them.
"""

from __future__ import annotations

import ctypes
import math
from array import array
from functools import lru_cache
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import FLOAT_DTYPES, INDEX_DTYPES, _DTYPE_CODE, _differentiated, _launch, _need_cuda, _need_dtype, _workspace

MAX_HEAD_DIM = 1024
_SCALINGS = (None, "linear", "ntk", "yarn")


def rope_frequencies(rotary_dim: int, *, theta: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                     original_length: int | None = None, fast_turns: float = 32.0, slow_turns: float = 1.0,
                     device: torch.device | str = "cuda") -> tuple[torch.Tensor, float]:
    """``(frequencies, scale)`` for ``rope`` / ``qk_norm_rope``: float64 ``[rotary_dim / 2]`` radians per position,
    ``theta ** (-2 i / rotary_dim)``, and the factor that the rotated part is multiplied with (1 but for ``"yarn"``).

    ``scaling`` stretches a context of ``original_length`` by ``factor``:

    * ``"linear"``  every frequency divided by ``factor`` (positions are interpolated);
    * ``"ntk"``     ``theta`` times ``factor ** (rotary_dim / (rotary_dim - 2))``: the slowest frequency is
      interpolated in full, the fastest not at all;
    * ``"yarn"``    by bands (Peng et al., 2023): frequencies that turn more than ``fast_turns`` times over
      ``original_length`` stay, those below ``slow_turns`` are interpolated, a ramp in between;
      ``scale = 1 + 0.1 ln(factor)``."""
    rotary_dim = int(rotary_dim)
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and not negative.")
    if not (theta > 0 and math.isfinite(theta)):
        raise ValueError("theta must be positive and finite.")
    if scaling not in _SCALINGS:
        raise ValueError(f"scaling must be one of None, 'linear', 'ntk', 'yarn'; got {scaling!r}.")
    if scaling is not None and not (factor >= 1 and math.isfinite(factor)):
        raise ValueError("factor must be finite and at least 1.")
    index = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    scale = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    frequencies = float(theta) ** (-index / max(rotary_dim, 1))
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "yarn":
        if original_length is None or original_length < 1:
            raise ValueError("scaling 'yarn' needs original_length, the context that the frequencies were trained for.")
        if not fast_turns > slow_turns:
            raise ValueError("fast_turns must exceed slow_turns.")
        turns = original_length * frequencies / (2.0 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        frequencies = frequencies * (keep + (1.0 - keep) / factor)
        scale = 1.0 + 0.1 * math.log(factor)
    return frequencies.to(device), scale


# ----------------------------------------------------------------------------------------------
# checks
# ----------------------------------------------------------------------------------------------
def _check_heads(name: str, x: torch.Tensor) -> None:
    _need_cuda(name, x)
    _need_dtype(name, x, FLOAT_DTYPES)
    if x.dim() not in (3, 4):
        raise ValueError(f"{name} must be shaped (batch, seq, heads, dim) or (tokens, heads, dim).")
    if not 1 <= x.shape[-1] <= MAX_HEAD_DIM:
        raise ValueError(f"{name} must have a head dimension between 1 and {MAX_HEAD_DIM}; got {x.shape[-1]}.")


def _check_positions(shape: torch.Size, device: torch.device, positions: torch.Tensor, frequencies: torch.Tensor) -> None:
    _need_cuda("positions", positions)
    _need_cuda("frequencies", frequencies)
    _need_dtype("positions", positions, INDEX_DTYPES)
    _need_dtype("frequencies", frequencies, (torch.float64,))
    lead = shape[:-2]
    if positions.shape != lead and positions.shape != lead[-1:]:
        wanted = f"{tuple(lead)}" + (f" or {tuple(lead[-1:])}" if len(lead) == 2 else "")
        raise ValueError(f"Shape mismatch: positions has shape {tuple(positions.shape)}, expected {wanted}.")
    if frequencies.dim() != 1 or 2 * frequencies.shape[0] > shape[-1]:
        raise ValueError(f"Shape mismatch: frequencies has shape {tuple(frequencies.shape)}, expected 1D with at most "
                         f"{shape[-1] // 2} entries (half the head dimension).")
    if not frequencies.is_contiguous():
        raise ValueError("frequencies must be contiguous.")
    for name, t in (("positions", positions), ("frequencies", frequencies)):
        if t.device != device:
            raise ValueError(f"Device mismatch: {name} is on {t.device}, the heads are on {device}.")


def _rows_readable(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself if its last dimension is contiguous, else a contiguous copy."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _heads_like(x: torch.Tensor) -> torch.Tensor:
    """An output of ``x``'s shape whose last dimension is contiguous, as the kernels write it: in ``x``'s layout where that
    is dense. Of an overlapping view (``unfold``) ``empty_like`` may order the dimensions otherwise."""
    out = torch.empty_like(x)
    return out if out.stride(-1) == 1 or x.shape[-1] == 1 else x.new_empty(x.shape)


# ----------------------------------------------------------------------------------------------
# what crosses the C ABI
# ----------------------------------------------------------------------------------------------
_NO_TENSOR = (0, 0, 0, 0)


def _placed(x: torch.Tensor) -> tuple[int, int, int, int]:
    """Pointer and element strides of (batch, seq, head)."""
    s = x.stride()
    return (x.data_ptr(), s[0], s[1], s[2]) if len(s) == 4 else (x.data_ptr(), 0, s[0], s[1])


def _row_fields(x: torch.Tensor, out: torch.Tensor, grad: torch.Tensor | None = None, weight: torch.Tensor | None = None,
                dweight: torch.Tensor | None = None) -> tuple[int, ...]:
    """The fields of ``lce_head_rows``, 64 bits each."""
    return (*_placed(x), *_placed(out), *(_NO_TENSOR if grad is None else _placed(grad)),
            0 if weight is None else weight.data_ptr(), 0 if dweight is None else dweight.data_ptr(), x.shape[-2])


_ROW_BYTES = ctypes.sizeof(_lib.HeadRows)


def _place(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor):
    """(batch, seq, dim, positions pointer, is int64, its batch stride, its seq stride, frequencies pointer, half)."""
    shape = x.shape
    stride = positions.stride()
    batch, seq, _, dim = shape if len(shape) == 4 else (1, *shape)
    return (batch, seq, dim, positions.data_ptr(), positions.dtype is torch.int64, stride[0] if len(stride) == 2 else 0,
            stride[-1], frequencies.data_ptr(), frequencies.shape[0])


# ----------------------------------------------------------------------------------------------
# rope
# ----------------------------------------------------------------------------------------------
def _rope(x, positions, frequencies, interleaved, scale, inverse):
    x = _rows_readable(x)
    out = _heads_like(x)
    rows = array("q", _row_fields(x, out))
    _launch("lce_rope", x.device, rows.buffer_info()[0], *_place(x, positions, frequencies), interleaved, scale, inverse,
            _DTYPE_CODE[x.dtype])
    return out


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, positions, frequencies, interleaved, scale, inverse):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (interleaved, scale, inverse)
        return _rope(x, positions, frequencies, interleaved, scale, inverse)

    @staticmethod
    def backward(ctx: Any, *grad_outputs):
        interleaved, scale, inverse = ctx.how
        # the rotation's transpose is the rotation by the negative angle, which is differentiable in turn
        turn = _Rope.apply if torch.is_grad_enabled() else _rope
        dx = turn(grad_outputs[0], *ctx.saved_tensors, interleaved, scale, not inverse)
        return dx, None, None, None, None, None


def rope(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *, interleaved: bool = False,
         scale: float = 1.0) -> torch.Tensor:
    """Rotate the first ``2 * len(frequencies)`` elements of every head of ``x`` by the angles
    ``positions * frequencies``; the other elements pass through.

    ``x`` is ``[batch, seq, heads, dim]`` or ``[tokens, heads, dim]``; ``positions`` int32 / int64, one per token
    (or ``[seq]`` for all sequences); ``frequencies`` float64, as ``rope_frequencies`` makes them. The pairs are
    ``(x[i], x[half + i])``, or ``(x[2i], x[2i + 1])`` with ``interleaved``; ``scale`` multiplies the rotated part.
    Differentiable in ``x``; the backward pass is the same kernel turning the other way."""
    _check_heads("x", x)
    _check_positions(x.shape, x.device, positions, frequencies)
    if _differentiated(x):
        return _Rope.apply(x, positions, frequencies, bool(interleaved), float(scale), False)
    return _rope(x, positions, frequencies, bool(interleaved), float(scale), False)


# ----------------------------------------------------------------------------------------------
# qk_norm_rope
# ----------------------------------------------------------------------------------------------
def _qk_forward(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale):
    q_out, k_out = _heads_like(q), _heads_like(k)
    rows = array("q", _row_fields(q, q_out, None, q_weight) + _row_fields(k, k_out, None, k_weight))
    at = rows.buffer_info()[0]
    _launch("lce_qk_norm_rope_forward", q.device, at, at + _ROW_BYTES, *_place(q, positions, frequencies), interleaved, scale,
            eps, _DTYPE_CODE[q.dtype])
    return q_out, k_out


@lru_cache(maxsize=None)
def _backward_bytes(dim: int) -> int:
    return _lib.lib().lce_qk_norm_rope_backward_workspace_bytes(dim)


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, frequencies)
        ctx.how = (eps, interleaved, scale)
        return _qk_forward(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, *grad_outputs):
        q, k, q_weight, k_weight, positions, frequencies = ctx.saved_tensors
        eps, interleaved, scale = ctx.how
        gq, gk = (_rows_readable(g) for g in grad_outputs)
        dq, dk = _heads_like(q), _heads_like(k)
        dqw = torch.empty_like(q_weight) if ctx.needs_input_grad[2] else None
        dkw = torch.empty_like(k_weight) if ctx.needs_input_grad[3] else None
        ws = _workspace(_backward_bytes(q.shape[-1]), q.device)
        rows = array("q", _row_fields(q, dq, gq, q_weight, dqw) + _row_fields(k, dk, gk, k_weight, dkw))
        at = rows.buffer_info()[0]
        _launch("lce_qk_norm_rope_backward", q.device, at, at + _ROW_BYTES, *_place(q, positions, frequencies), interleaved,
                scale, eps, _DTYPE_CODE[q.dtype], ws.data_ptr(), ws.numel())
        need = ctx.needs_input_grad
        return (dq if need[0] else None), (dk if need[1] else None), dqw, dkw, None, None, None, None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                 frequencies: torch.Tensor, *, eps: float = 1e-6, interleaved: bool = False,
                 scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """``(rope(norm(q) * q_weight), rope(norm(k) * k_weight))`` in one launch, where ``norm`` divides every head by
    its root mean square over ``dim`` (``rmsnorm`` over one head).

    ``q`` is ``[batch, seq, heads, dim]``, ``k`` ``[batch, seq, kv_heads, dim]`` (or both without ``batch``), the
    weights are ``[dim]``; ``positions``, ``frequencies``, ``interleaved`` and ``scale`` as for ``rope``. Nothing is
    rounded between the norm and the rotation. Differentiable in ``q``, ``k`` and the weights: the backward pass reads
    the gradients and the inputs once; the weights' gradients are summed in a fixed order."""
    _check_heads("q", q)
    _check_heads("k", k)
    shape, dtype, device = q.shape, q.dtype, q.device
    dim = shape[-1]
    if k.shape[:-2] != shape[:-2] or k.shape[-1] != dim:
        raise ValueError(f"Shape mismatch: k has shape {tuple(k.shape)}, q has shape {tuple(shape)}; they may differ in "
                         "the number of heads only.")
    for name, t in (("k", k), ("q_weight", q_weight), ("k_weight", k_weight)):
        if t.device != device:
            raise ValueError(f"Device mismatch: {name} is on {t.device}, q is on {device}.")
        if t.dtype != dtype:
            raise ValueError(f"Dtype mismatch: {name} has dtype {t.dtype}, q has dtype {dtype}.")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t.shape != (dim,):
            raise ValueError(f"Shape mismatch: {name} has shape {tuple(t.shape)}, expected ({dim},).")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous.")
    _check_positions(shape, device, positions, frequencies)
    if not eps >= 0:
        raise ValueError("eps must not be negative.")
    q, k = _rows_readable(q), _rows_readable(k)
    if _differentiated(q, k, q_weight, k_weight):
        return _QKNormRope.apply(q, k, q_weight, k_weight, positions, frequencies, float(eps), bool(interleaved), float(scale))
    return _qk_forward(q, k, q_weight, k_weight, positions, frequencies, float(eps), bool(interleaved), float(scale))
