"""sample_logits on the sizes at which the call changes its form: rows whose share per CTA no longer fits shared memory,
batches without a filter, rows of more chunks than the form with a bin per value has room for. GPU only."""

from __future__ import annotations

import pytest
import torch

import helion_b200
from test_gpu_sample import _check, _gen, _logits

pytestmark = pytest.mark.gpu
DEV = "cuda"


# eight CTAs a row keep 160 KB each: 327680 logits in 32 bits, 655360 in 16
@pytest.mark.parametrize(("dtype", "vocab"), [(torch.float32, 327680), (torch.float32, 327681), (torch.float32, 400003),
                                              (torch.float16, 655361), (torch.float16, 700001), (torch.bfloat16, 700001)])
@pytest.mark.parametrize("filters", [dict(), dict(top_k=50), dict(top_k=30000, top_p=0.9), dict(top_p=0.95), dict(temperature=0),
                                     dict(temperature=1.2, top_k=5000, min_p=0.001)])
def test_rows_beyond_shared_memory(dtype, vocab, filters):
    logits = _logits(2, vocab, dtype, vocab, masked=0.1)
    _check(logits, torch.rand(2, generator=_gen(3), device=DEV), **filters)


@pytest.mark.parametrize("vocab", [32767, 32768, 32771])
@pytest.mark.parametrize("filters", [dict(), dict(min_p=0.02), dict(temperature=0.5), dict(temperature=0)])
def test_batches_without_a_rank_filter(vocab, filters):
    logits = _logits(128, vocab, torch.bfloat16, vocab)
    _check(logits, torch.rand(128, generator=_gen(5), device=DEV), **filters)


@pytest.mark.parametrize("vocab", [1048560, 1048577])  # 1024 chunks of 1024 logits, and one more
def test_more_chunks_than_a_row_has_room_for(vocab):
    logits = _logits(40, vocab, torch.bfloat16, 9)
    u = torch.rand(40, generator=_gen(6), device=DEV)
    u[0], u[39] = 0.0, 1.0
    whole = _check(logits[:3], u[:3], top_p=0.9)  # three rows take the cluster form
    token, logprob = helion_b200.sample_logits(logits, u, top_p=0.9, return_logprob=True)
    assert torch.equal(token[:3], whole[0])
    assert bool(((logprob[:3] - whole[1]).abs() <= 2.0 ** -22 * whole[1].abs() + 1e-9).all())
    last = _check(logits[39:], u[39:], top_p=0.9)
    assert int(last[0][0]) == int(token[39])
