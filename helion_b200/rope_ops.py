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

import math
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import FLOAT_DTYPES, INDEX_DTYPES, _DTYPE_CODE, _need_cuda, _need_dtype, _on_device, _stream, _workspace

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


def _check_positions(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor) -> None:
    _need_cuda("positions", positions)
    _need_cuda("frequencies", frequencies)
    _need_dtype("positions", positions, INDEX_DTYPES)
    _need_dtype("frequencies", frequencies, (torch.float64,))
    lead = x.shape[:-2]
    if positions.shape != lead and positions.shape != lead[-1:]:
        wanted = f"{tuple(lead)}" + (f" or {tuple(lead[-1:])}" if len(lead) == 2 else "")
        raise ValueError(f"Shape mismatch: positions has shape {tuple(positions.shape)}, expected {wanted}.")
    if frequencies.dim() != 1 or 2 * frequencies.shape[0] > x.shape[-1]:
        raise ValueError(f"Shape mismatch: frequencies has shape {tuple(frequencies.shape)}, expected 1D with at most "
                         f"{x.shape[-1] // 2} entries (half the head dimension).")
    if not frequencies.is_contiguous():
        raise ValueError("frequencies must be contiguous.")
    for name, t in (("positions", positions), ("frequencies", frequencies)):
        if t.device != x.device:
            raise ValueError(f"Device mismatch: {name} is on {t.device}, the heads are on {x.device}.")


def _rows_readable(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself if its last dimension is contiguous, else a contiguous copy."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _strides(x: torch.Tensor) -> tuple[int, int, int]:
    """Element strides of (batch, seq, head); a dimension of one entry has none (0)."""
    shape, stride = x.shape, x.stride()
    head = stride[-2] if shape[-2] > 1 else 0
    seq = stride[-3] if shape[-3] > 1 else 0
    return (stride[0] if len(shape) == 4 and shape[0] > 1 else 0), seq, head


_NO_STRIDES = (0, 0, 0)


def _rows(x: torch.Tensor, out: torch.Tensor, grad: torch.Tensor | None = None, weight: torch.Tensor | None = None,
          dweight: torch.Tensor | None = None) -> _lib.HeadRows:
    return _lib.HeadRows(x.data_ptr(), _strides(x), out.data_ptr(), _strides(out),
                         None if grad is None else grad.data_ptr(), _NO_STRIDES if grad is None else _strides(grad),
                         None if weight is None else weight.data_ptr(), None if dweight is None else dweight.data_ptr(),
                         x.shape[-2])


def _place(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor):
    """(batch, seq, dim, positions pointer, is int64, its batch stride, its seq stride, frequencies pointer, half)."""
    shape = x.shape
    batch, seq = (1, shape[0]) if len(shape) == 3 else (shape[0], shape[1])
    stride = positions.stride()
    return (batch, seq, shape[-1], positions.data_ptr(), int(positions.dtype == torch.int64),
            stride[0] if len(stride) == 2 else 0, stride[-1], frequencies.data_ptr(), frequencies.shape[0])


# ----------------------------------------------------------------------------------------------
# rope
# ----------------------------------------------------------------------------------------------
def _rope(x, positions, frequencies, interleaved, scale, inverse):
    x = _rows_readable(x)
    out = torch.empty_like(x)
    dev = x.device
    with _on_device(dev):
        _lib.check(
            _lib.lib().lce_rope(_rows(x, out), *_place(x, positions, frequencies), int(interleaved), scale, int(inverse),
                                _DTYPE_CODE[x.dtype], _stream(dev)),
            "lce_rope",
        )
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
        dx = _Rope.apply(grad_outputs[0], *ctx.saved_tensors, interleaved, scale, not inverse)
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
    _check_positions(x, positions, frequencies)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Rope.apply(x, positions, frequencies, bool(interleaved), float(scale), False)
    return _rope(x, positions, frequencies, interleaved, float(scale), False)


# ----------------------------------------------------------------------------------------------
# qk_norm_rope
# ----------------------------------------------------------------------------------------------
def _qk_forward(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale):
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    dev = q.device
    with _on_device(dev):
        _lib.check(
            _lib.lib().lce_qk_norm_rope_forward(_rows(q, q_out, weight=q_weight), _rows(k, k_out, weight=k_weight),
                                                *_place(q, positions, frequencies), int(interleaved), scale, eps,
                                                _DTYPE_CODE[q.dtype], _stream(dev)),
            "lce_qk_norm_rope_forward",
        )
    return q_out, k_out


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
        dq, dk = torch.empty_like(q), torch.empty_like(k)
        dqw = torch.empty_like(q_weight) if ctx.needs_input_grad[2] else None
        dkw = torch.empty_like(k_weight) if ctx.needs_input_grad[3] else None
        dev = q.device
        L = _lib.lib()
        ws = _workspace(L.lce_qk_norm_rope_backward_workspace_bytes(q.shape[-1]), dev)
        with _on_device(dev):
            _lib.check(
                L.lce_qk_norm_rope_backward(_rows(q, dq, gq, q_weight, dqw), _rows(k, dk, gk, k_weight, dkw),
                                            *_place(q, positions, frequencies), int(interleaved), scale, eps,
                                            _DTYPE_CODE[q.dtype], ws.data_ptr(), ws.numel(), _stream(dev)),
                "lce_qk_norm_rope_backward",
            )
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
    if k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"Shape mismatch: k has shape {tuple(k.shape)}, q has shape {tuple(q.shape)}; they may differ in "
                         "the number of heads only.")
    dim = q.shape[-1]
    for name, t in (("k", k), ("q_weight", q_weight), ("k_weight", k_weight)):
        if t.device != q.device:
            raise ValueError(f"Device mismatch: {name} is on {t.device}, q is on {q.device}.")
        if t.dtype != q.dtype:
            raise ValueError(f"Dtype mismatch: {name} has dtype {t.dtype}, q has dtype {q.dtype}.")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if tuple(t.shape) != (dim,):
            raise ValueError(f"Shape mismatch: {name} has shape {tuple(t.shape)}, expected ({dim},).")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous.")
    _check_positions(q, positions, frequencies)
    if not eps >= 0:
        raise ValueError("eps must not be negative.")
    q, k = _rows_readable(q), _rows_readable(k)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad or k_weight.requires_grad):
        return _QKNormRope.apply(q, k, q_weight, k_weight, positions, frequencies, float(eps), bool(interleaved), float(scale))
    return _qk_forward(q, k, q_weight, k_weight, positions, frequencies, float(eps), interleaved, float(scale))
