"""sample_logits on the host: refusals and the C ABI's checks. No kernel is launched here."""

from __future__ import annotations

import pytest
import torch

import helion_b200
from helion_b200 import _lib, decode_ops


@pytest.fixture()
def any_device(monkeypatch):
    monkeypatch.setattr(decode_ops, "_need_cuda", lambda name, t: None)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="logits must be a CUDA tensor."):
        helion_b200.sample_logits(torch.randn(2, 8), torch.rand(2))


@pytest.mark.parametrize(("change", "message"), [
    (dict(logits=torch.randn(2, 8).double()), "logits must have one of these dtypes"),
    (dict(logits=torch.tensor(1.0)), "logits must have at least 1 dimension"),
    (dict(logits=torch.randn(2, 0)), "vocab_size must be positive"),
    (dict(uniforms=torch.rand(2).double()), "uniforms must have one of these dtypes: float32."),
    (dict(uniforms=torch.rand(3)), r"uniforms has shape \(3,\), expected \(2,\)."),
    (dict(uniforms=torch.rand(2, 1)), r"uniforms has shape \(2, 1\)"),
    (dict(temperature=-0.5), "temperature must be >= 0"),
    (dict(temperature=float("nan")), "temperature must be >= 0"),
    (dict(temperature=float("inf")), "temperature must be >= 0 and finite"),
    (dict(temperature=torch.ones(2).double()), "temperature must have one of these dtypes: float32."),
    (dict(temperature=torch.ones(1)), r"temperature has shape \(1,\), expected \(2,\)."),
    (dict(top_k=-1), "top_k must be >= 0"),
    (dict(top_k=torch.ones(2)), "top_k must have one of these dtypes: int32, int64."),
    (dict(top_p=0.0), "top_p must satisfy"),
    (dict(top_p=1.5), "top_p must satisfy"),
    (dict(min_p=-0.1), "min_p must satisfy"),
    (dict(min_p=1.1), "min_p must satisfy"),
    (dict(min_p=torch.ones(2, 2)), r"min_p has shape \(2, 2\)"),
])
def test_refusals(any_device, change, message):
    args = dict(logits=torch.randn(2, 8), uniforms=torch.rand(2)) | change
    logits, uniforms = args.pop("logits"), args.pop("uniforms")
    with pytest.raises(ValueError, match=message):
        helion_b200.sample_logits(logits, uniforms, **args)


def test_c_abi_refuses_before_it_touches_a_device():
    L = _lib.lib()
    p = 256

    def call(logits=p, ld=100, rows=2, vocab=100, dtype=0, uniform=p, token=p, ws=None, ws_bytes=1 << 40):
        return L.lce_sample_logits(logits, ld, rows, vocab, dtype, uniform, None, 1.0, None, 0, 0, None, 1.0, None, 0.0, token,
                                   None, ws, ws_bytes, None)

    assert call(dtype=7) == 1 and call(rows=-1) == 1 and call(vocab=0) == 1 and call(ld=99) == 1
    assert call(logits=None) == 1 and call(uniform=None) == 1 and call(token=None) == 1
    assert call(vocab=1 << 31, ld=1 << 31) == 6 and call(rows=1 << 31) == 6
    assert call(rows=0) == 0
