"""rope / qk_norm_rope on the host: refusals, the frequency schedules, and the struct that crosses the C ABI. No kernel
is launched here."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import helion_b200
from helion_b200 import _lib, rope_ops


@pytest.fixture()
def any_device(monkeypatch):
    monkeypatch.setattr(rope_ops, "_need_cuda", lambda name, t: None)


def _good(batch=2, seq=3, heads=4, kv=2, dim=16):
    return dict(q=torch.randn(batch, seq, heads, dim), k=torch.randn(batch, seq, kv, dim), q_weight=torch.ones(dim),
                k_weight=torch.ones(dim), positions=torch.zeros(batch, seq, dtype=torch.int64),
                frequencies=torch.ones(dim // 2, dtype=torch.float64))


def test_cpu_tensors_are_refused():
    a = _good()
    with pytest.raises(ValueError, match="x must be a CUDA tensor."):
        helion_b200.rope(a["q"], a["positions"], a["frequencies"])
    with pytest.raises(ValueError, match="q must be a CUDA tensor."):
        helion_b200.qk_norm_rope(**a)


@pytest.mark.parametrize(("change", "message"), [
    (dict(x=torch.randn(3, 16)), r"x must be shaped \(batch, seq, heads, dim\) or \(tokens, heads, dim\)"),
    (dict(x=torch.randn(2, 3, 4, 16).double()), "x must have one of these dtypes"),
    (dict(x=torch.randn(2, 3, 4, 0)), "head dimension between 1 and 1024; got 0"),
    (dict(x=torch.randn(1, 1, 1, 1025)), "head dimension between 1 and 1024; got 1025"),
    (dict(positions=torch.zeros(2, 3)), "positions must have one of these dtypes: int32, int64."),
    (dict(positions=torch.zeros(2, 4, dtype=torch.int64)), r"positions has shape \(2, 4\), expected \(2, 3\) or \(3,\)."),
    (dict(positions=torch.zeros(2, dtype=torch.int64)), r"positions has shape \(2,\), expected"),
    (dict(frequencies=torch.ones(8)), "frequencies must have one of these dtypes: float64."),
    (dict(frequencies=torch.ones(9, dtype=torch.float64)), "at most 8 entries"),
    (dict(frequencies=torch.ones(2, 4, dtype=torch.float64)), r"frequencies has shape \(2, 4\)"),
    (dict(frequencies=torch.ones(16, dtype=torch.float64)[::2]), "frequencies must be contiguous."),
])
def test_rope_refusals(any_device, change, message):
    a = _good()
    args = dict(x=a["q"], positions=a["positions"], frequencies=a["frequencies"]) | change
    with pytest.raises(ValueError, match=message):
        helion_b200.rope(args["x"], args["positions"], args["frequencies"])


@pytest.mark.parametrize(("change", "message"), [
    (dict(k=torch.randn(2, 4, 2, 16)), "may differ in the number of heads only"),
    (dict(k=torch.randn(2, 3, 2, 8)), "may differ in the number of heads only"),
    (dict(k=torch.randn(3, 2, 16)), "may differ in the number of heads only"),
    (dict(k=torch.randn(2, 3, 2, 16).half()), "Dtype mismatch: k has dtype torch.float16"),
    (dict(q_weight=torch.ones(8)), r"q_weight has shape \(8,\), expected \(16,\)."),
    (dict(k_weight=torch.ones(16).half()), "Dtype mismatch: k_weight"),
    (dict(k_weight=torch.ones(32)[::2]), "k_weight must be contiguous."),
    (dict(eps=-1.0), "eps must not be negative."),
    (dict(eps=float("nan")), "eps must not be negative."),
])
def test_qk_norm_rope_refusals(any_device, change, message):
    with pytest.raises(ValueError, match=message):
        helion_b200.qk_norm_rope(**(_good() | change))


def test_frequencies():
    f, scale = helion_b200.rope_frequencies(8, theta=100.0, device="cpu")
    assert f.dtype == torch.float64 and scale == 1.0
    torch.testing.assert_close(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15, atol=0)
    linear, _ = helion_b200.rope_frequencies(8, theta=100.0, scaling="linear", factor=4.0, device="cpu")
    torch.testing.assert_close(linear, f / 4, rtol=1e-15, atol=0)
    ntk, _ = helion_b200.rope_frequencies(8, theta=100.0, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and abs(float(ntk[-1] / (f[-1] / 4)) - 1) < 1e-14  # the ends: untouched, interpolated in full
    # by bands: original_length * f / 2 pi turns; above `fast` kept, below `slow` divided, half-way the mean
    f2, _ = helion_b200.rope_frequencies(64, device="cpu")
    length = 4096
    yarn, scale = helion_b200.rope_frequencies(64, scaling="yarn", factor=8.0, original_length=length, device="cpu")
    turns = length * f2 / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], f2[turns >= 32])
    torch.testing.assert_close(yarn[turns <= 1], f2[turns <= 1] / 8, rtol=1e-15, atol=0)
    inside = (turns > 1) & (turns < 32)
    assert inside.any() and bool((yarn[inside] < f2[inside]).all() and (yarn[inside] > f2[inside] / 8).all())
    assert scale == 1.0 + 0.1 * math.log(8.0)
    assert helion_b200.rope_frequencies(0, device="cpu")[0].shape == (0,)


@pytest.mark.parametrize(("kw", "message"), [
    (dict(rotary_dim=7), "rotary_dim must be even"),
    (dict(rotary_dim=-2), "rotary_dim must be even"),
    (dict(rotary_dim=8, theta=0.0), "theta must be positive"),
    (dict(rotary_dim=8, theta=float("inf")), "theta must be positive and finite"),
    (dict(rotary_dim=8, scaling="cubic"), "scaling must be one of"),
    (dict(rotary_dim=8, scaling="linear", factor=0.5), "factor must be finite and at least 1"),
    (dict(rotary_dim=8, scaling="yarn", factor=2.0), "needs original_length"),
    (dict(rotary_dim=8, scaling="yarn", factor=2.0, original_length=64, fast_turns=1.0), "fast_turns must exceed"),
])
def test_frequency_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        helion_b200.rope_frequencies(**kw, device="cpu")


def test_c_abi_refuses_before_it_touches_a_device():
    L = _lib.lib()
    assert ctypes.sizeof(_lib.HeadRows) == 15 * 8
    rows = _lib.HeadRows(16, (64, 32, 8), 16, (64, 32, 8), None, (0, 0, 0), 16, None, 4)
    pos, freq = 16, 16  # never dereferenced: every call here is refused

    def rope(r=rows, batch=1, seq=1, dim=8, positions=pos, frequencies=freq, half=4, dtype=0):
        return L.lce_rope(None if r is None else ctypes.byref(r), batch, seq, dim, positions, 1, 0, 1, frequencies, half, 0, 1.0, 0, dtype, None)

    assert rope(dtype=9) == 1 and rope(batch=-1) == 1 and rope(half=5) == 1 and rope(dim=0) == 1
    assert rope(dim=1025) == 6 and rope(batch=1 << 40) == 6
    assert rope(positions=None) == 1 and rope(frequencies=None) == 1 and rope(r=None) == 1
    assert rope(r=_lib.HeadRows(None, (64, 32, 8), 16, (64, 32, 8), None, (0, 0, 0), None, None, 4)) == 1
    assert rope(r=_lib.HeadRows(16, (0, 0, 0), 16, (0, 0, 0), None, (0, 0, 0), None, None, -1)) == 1
    assert rope(batch=0) == 0  # nothing to do
    need = L.lce_qk_norm_rope_backward_workspace_bytes(8)
    assert need > 0 and L.lce_qk_norm_rope_backward_workspace_bytes(0) == 0
    back = _lib.HeadRows(16, (64, 32, 8), 16, (64, 32, 8), 16, (64, 32, 8), 16, 16, 4)
    args = (1, 1, 8, pos, 1, 0, 1, freq, 4, 0, 1.0, 1e-6, 0)
    assert L.lce_qk_norm_rope_backward(ctypes.byref(back), ctypes.byref(back), *args, 16, need - 1, None) == 3
    assert L.lce_qk_norm_rope_backward(ctypes.byref(back), ctypes.byref(back), *args, None, need, None) == 3
    assert L.lce_qk_norm_rope_backward(ctypes.byref(rows), ctypes.byref(back), *args, 16, need, None) == 1  # no gradient
    assert L.lce_qk_norm_rope_forward(ctypes.byref(rows), None, *args, None) == 1
