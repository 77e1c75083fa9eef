"""Scratch while a stream is captured: the stream that counts is the one of the tensors' device. Two devices are played by
fakes of torch's queries, so that no GPU is needed."""

from __future__ import annotations

from contextlib import contextmanager

import pytest
import torch

from helion_b200 import ops


@pytest.fixture
def two_devices(monkeypatch):
    """A state whose 'current' is the current device and whose 'captured' is the device whose stream is being captured."""
    state = {"current": 0, "captured": None}

    @contextmanager
    def device(d):
        previous, state["current"] = state["current"], torch.device(d).index
        try:
            yield
        finally:
            state["current"] = previous

    monkeypatch.setattr(ops, "_current_device", lambda: state["current"])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "_stream_capturing", lambda: state["current"] == state["captured"])
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(ops, "_ws_cache", {})
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda n, dtype=None, device=None: empty(n, dtype=dtype))
    return state


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("captured", [None, 0, 1])
def test_scratch_of_a_captured_call_is_its_own(two_devices, monkeypatch, current, captured):
    device = torch.device("cuda", 0)
    two_devices.update(current=0, captured=None)
    cached = ops._workspace(1000, device)
    assert ops._workspace(1000, device) is cached
    two_devices.update(current=current, captured=captured)
    own = captured == 0  # the tensors' device
    assert ops._capturing(device) is own
    assert (ops._workspace(1000, device) is not cached) is own
    offered = []

    def call(what, device, *args):
        offered.append(args[-3])
        return ops._lib.ERR_WS_TOO_SMALL if args[-3] is None else 0

    monkeypatch.setattr(ops, "_call", call)
    ops._launch_scratch("anything", lambda: 1000, device, flags=0)
    assert (cached.data_ptr() not in offered) is own
    assert two_devices["current"] == current
