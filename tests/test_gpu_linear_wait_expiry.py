"""The bounded waits of linear's kernels are made to run out, and each launch must come back with a status code, not hang.

The limit is shortened to a few milliseconds and the producers announce 16 bytes more on their first barrier than their copies
deliver: every copy lands, the barrier never completes, no tensor-core instruction is issued and nothing is in flight when a
kernel exits. Nothing traps or faults; the same call gives the right result afterwards. GPU only."""

from __future__ import annotations

import pytest
import torch

import helion_b200
from helion_b200 import _lib
from oracle import block_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
LIMIT_NS = 3_000_000  # 3 ms


# a cluster of one CTA, of eight whose ring runs full, both over several tokens; a single-CTA tile; a pair of CTAs with eight
# epilogue warps
@pytest.mark.parametrize(("m", "k", "n"), [(1, 64, 128), (16, 4096, 256), (33, 4096, 256), (100, 64, 256), (256, 64, 256)])
def test_a_wait_runs_out_with_a_status_code_and_the_next_launch_is_fine(m, k, n):
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, k, generator=g).bfloat16().to(DEV)
    w = (torch.randn(n, k, generator=g) * k ** -0.5).bfloat16().to(DEV)
    b = torch.randn(n, generator=g).bfloat16().to(DEV)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    L = _lib.lib()
    _lib.check(L.lce_debug_wait_test(LIMIT_NS, 16), "lce_debug_wait_test")
    try:
        helion_b200.linear(x, w, b, activation="gelu")
        torch.cuda.synchronize()  # returns: the waits gave up after 3 ms each
        # whichever role's timer ran out first has its code in the word: producer 101, issuer 102, epilogue 103
        assert _lib.device_status() in (101, 102, 103)
        assert _lib.device_status() == 0  # read and cleared
    finally:
        _lib.check(L.lce_debug_wait_test(0, 0), "lce_debug_wait_test")
        _lib.device_status()
    y = helion_b200.linear(x, w, b, activation="gelu")
    ref, _ = block_oracle.linear(x, w, b, "gelu")
    torch.cuda.synchronize()
    # one rounding of the result, 2^-8; sums of k products in 32 bits, k 2^-24 of sum |x w| + |b| < 16 sqrt(k / 64)
    assert bool(((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (k + 1) * 2.0 ** -24 * 16 * (k / 64) ** 0.5 + 4e-6).all())
    assert _lib.device_status() == 0
