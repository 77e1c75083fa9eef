"""sample_logits on batches whose masked logits are large finite negatives (-1e4, the type's lowest) instead of -inf. GPU only.

Large bf16 batches count their values in bins, of which these have none. Tokens have to be equal to the definition's, as
everywhere; the log-probabilities are rounded once."""

from __future__ import annotations

import pytest
import torch

from helion_b200 import _lib
from test_gpu_sample import FILTERS, _check, _gen, _logits

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = float("inf")
LOWEST = torch.finfo(torch.bfloat16).min


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("mask", [-1016.0, -1020.0, -1024.0, -1e4, LOWEST])  # -1016 is the lowest bf16 value with a bin
def test_masks_of_every_size(dtype, mask):
    rows, vocab = 81, 32771
    mask = max(mask, torch.finfo(dtype).min)
    logits = _logits(rows, vocab, dtype, 41)
    g = _gen(42)

    def hidden(share):
        return torch.rand(vocab, generator=g, device=DEV) < share

    for at in range(0, rows, 9):  # every kind meets nine of the filters
        logits[at + 1].masked_fill_(hidden(0.2), mask)
        logits[at + 2, 5:] = mask  # fewer than most top_k
        logits[at + 3] = mask  # nothing else: all are equal
        logits[at + 4] -= 1000.0  # the maximum so low that masked logits weigh something, or nearly
        logits[at + 4].masked_fill_(hidden(0.2), mask)
        logits[at + 5].masked_fill_(hidden(0.3), -INF)
        logits[at + 5].masked_fill_(hidden(0.3), float("nan"))
        logits[at + 5].masked_fill_(hidden(0.3), mask)
        logits[at + 6, 7::9] = mask
        logits[at + 6, 11::1001] = 1e-12 if dtype == torch.bfloat16 else 3e-7  # and a value without a bin
        logits[at + 7] = -INF
        logits[at + 7, at::3001] = mask
        logits[at + 8, :-1] = mask
    u = torch.rand(rows, generator=_gen(43), device=DEV)
    u[1::9], u[2], u[5] = torch.linspace(0, 1, 9, device=DEV), 0.0, 1.0
    params = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    lists = {name: [FILTERS[(5 * i + i // 9) % len(FILTERS)].get(name, off) for i in range(rows)] for name, off in params.items()}
    first = _check(logits, u, **lists)
    second = _check(logits.clone(), u, **lists)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("filters", [dict(), dict(min_p=0.05), dict(temperature=3.0), dict(top_p=0.9), dict(top_k=30)])
def test_masked_batches_with_one_filter_for_all(filters):
    rows, vocab = 128, 32768
    logits = _logits(rows, vocab, torch.bfloat16, 51)
    logits.masked_fill_(torch.rand(rows, vocab, generator=_gen(52), device=DEV) < 0.2, -1e4)
    token, _ = _check(logits, torch.rand(rows, generator=_gen(53), device=DEV), **filters)
    assert bool((logits.gather(1, token[:, None]) > -1000).all())
