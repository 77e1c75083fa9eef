"""rope and qk_norm_rope against float64 definitions: layouts, head sizes, types, far positions, gradients, capture.
GPU only.

Tolerances, from arithmetic. A result is rounded once: half a unit, eps / 2 relative. Before that, in 32 bits:
an angle's fraction of a turn is rounded to 24 bits (2 pi x 0.5 x 2^-25 < 1e-7 in angle), cos and sin are good to a few
2^-24 (the hardware's, for 16-bit types, to 2^-21.2 = 4.2e-7), and the rotation adds three roundings: below 6e-7 of the pair's magnitudes (|a| + |b|, at most twice the row's
largest). A row's sum of squares of up to 1024 terms passes through at most 37 additions per lane and butterfly, 2.2e-6
relative, half of that in rstd, which adds 2e-7 of its own: 2e-6 of a normalised element. The backward combines
two such sums: 1e-5 of the magnitudes that it subtracts. dweight adds at most a few hundred terms in sequence:
1e-5 of the sum of their magnitudes."""

from __future__ import annotations

import ctypes

import pytest
import torch

import helion_b200
from helion_b200 import _lib
from oracle import block_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _close(got, ref, dtype, slack):
    assert got.dtype == dtype and got.shape == ref.shape
    info = torch.finfo(dtype)
    bound = (info.eps / 2) * ref.abs() * (1 + info.eps) + info.tiny * info.eps + slack
    worst = ((got.double() - ref).abs() - bound).max() if ref.numel() else torch.zeros(())
    assert worst <= 0, f"off by {float(worst):.3e} more than the bound"


def _rowmax(t):
    return t.abs().amax(-1, keepdim=True).double()


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _heads(layout, batch, seq, heads, dim, dtype, seed):
    g = _gen(seed)
    if layout == "bshd":
        return torch.randn(batch, seq, heads, dim, generator=g, device=DEV).to(dtype)
    if layout == "bhsd":  # a transposed view of [batch, heads, seq, dim]
        return torch.randn(batch, heads, seq, dim, generator=g, device=DEV).to(dtype).transpose(1, 2)
    if layout == "fused":  # a slice of a wider projection
        return torch.randn(batch, seq, heads + 3, dim, generator=g, device=DEV).to(dtype)[:, :, 2:2 + heads]
    if layout == "offset":  # rows that start off a 16-byte boundary
        flat = torch.randn(batch * seq * heads * dim + 1, generator=g, device=DEV).to(dtype)
        return flat[1:].view(batch, seq, heads, dim)
    if layout == "lastdim":  # the last dimension is not contiguous
        return torch.randn(batch, seq, dim, heads, generator=g, device=DEV).to(dtype).transpose(2, 3)
    raise AssertionError(layout)


SHAPES = [  # dim, rotary, interleaved
    (128, 128, False), (128, 128, True), (128, 64, False), (64, 64, False), (80, 32, True), (80, 32, False), (72, 36, False),
    (72, 36, True), (72, 18, False), (256, 256, False), (512, 512, True), (512, 256, False), (1024, 1024, False), (1, 0, False),
    (7, 6, False), (7, 4, True), (40, 8, True), (24, 24, False), (16, 0, False), (8, 2, True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("dim", "rotary", "interleaved"), SHAPES)
def test_rope_forward_and_gradient(dtype, dim, rotary, interleaved):
    batch, seq, heads = 2, 5, 3
    x = _heads("bshd", batch, seq, heads, dim, dtype, dim + rotary).requires_grad_(True)
    pos = torch.randint(0, 5000, (batch, seq), generator=_gen(1), device=DEV)
    freq, _ = helion_b200.rope_frequencies(rotary)
    y = helion_b200.rope(x, pos, freq, interleaved=interleaved, scale=1.25)
    ref = block_oracle.rope(x.detach(), pos, freq, interleaved, 1.25)
    _close(y.detach(), ref, dtype, 6e-7 * 2 * 1.25 * _rowmax(x.detach()))
    assert torch.equal(y.detach()[..., rotary:], x.detach()[..., rotary:])  # what is not rotated passes through
    dy = _heads("bshd", batch, seq, heads, dim, dtype, 7)
    (dx,) = torch.autograd.grad(y, x, dy)
    _close(dx, block_oracle.rope(dy, pos, freq, interleaved, 1.25, inverse=True), dtype, 6e-7 * 2 * 1.25 * _rowmax(dy))


@pytest.mark.parametrize("layout", ["bshd", "bhsd", "fused", "offset", "lastdim"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("batch", "seq", "heads"), [(1, 1, 1), (3, 1, 40), (2, 130, 5), (1, 700, 8)])
def test_layouts_and_lengths(layout, dtype, batch, seq, heads):
    dim = 64
    x = _heads(layout, batch, seq, heads, dim, dtype, 3)
    freq, _ = helion_b200.rope_frequencies(dim)
    pos = torch.arange(seq, device=DEV, dtype=torch.int32) + 11
    ref = block_oracle.rope(x, pos.expand(batch, seq), freq)
    y = helion_b200.rope(x, pos, freq)  # one [seq] vector for all sequences
    _close(y, ref, dtype, 1.2e-6 * _rowmax(x))
    assert torch.equal(y, helion_b200.rope(x, pos.long().expand(batch, seq), freq))
    if layout == "bhsd":
        assert y.transpose(1, 2).is_contiguous()  # a dense permuted input keeps its layout
    if batch == 1:  # [tokens, heads, dim]
        assert torch.equal(helion_b200.rope(x[0], pos, freq), y[0])
        assert torch.equal(helion_b200.rope(x[0], torch.stack([pos, pos], 1)[:, 0], freq), y[0])  # positions with a stride


@pytest.mark.parametrize("far", [0, -3, 123456, (1 << 24) + 1, (1 << 31) + 5, 1 << 40])
def test_far_positions_keep_their_angle(far):
    x = torch.randn(1, 4, 2, 32, generator=_gen(5), device=DEV)
    freq, _ = helion_b200.rope_frequencies(32)
    pos = far + torch.arange(4, device=DEV)[None]
    # the product's 53 bits leave far * 2^-53 of absolute error in the angle on each side
    slack = (1.2e-6 + 4 * abs(far) * 2.0 ** -53) * _rowmax(x)
    _close(helion_b200.rope(x, pos, freq), block_oracle.rope(x, pos, freq), torch.float32, slack)


def test_empty_inputs_and_no_heads():
    freq, _ = helion_b200.rope_frequencies(16)
    for shape, pos in (((0, 4, 2, 16), (0, 4)), ((2, 0, 2, 16), (2, 0)), ((2, 3, 0, 16), (2, 3)), ((0, 2, 16), (0,))):
        x = torch.randn(shape, device=DEV, requires_grad=True)
        y = helion_b200.rope(x, torch.zeros(pos, dtype=torch.int64, device=DEV), freq)
        assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    q = torch.randn(0, 2, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    k = torch.randn(0, 1, 16, device=DEV)
    out = helion_b200.qk_norm_rope(q, k, w, w, torch.zeros(0, dtype=torch.int64, device=DEV), freq)
    (dw,) = torch.autograd.grad(out[0].sum() + out[1].sum(), w)
    assert torch.equal(dw, torch.zeros_like(dw))  # a sum of nothing


def test_values_that_are_not_finite_stay_in_their_row():
    x = torch.randn(1, 6, 4, 128, generator=_gen(2), device=DEV).bfloat16()
    x[0, 2, 1, 5], x[0, 3, 0, 100], x[0, 4, 3, 0] = float("nan"), float("inf"), float("-inf")
    freq, _ = helion_b200.rope_frequencies(64)
    pos = torch.arange(6, device=DEV)
    w = torch.ones(128, device=DEV, dtype=torch.bfloat16)
    y = helion_b200.rope(x, pos, freq)
    q, k = helion_b200.qk_norm_rope(x, x, w, w, pos, freq)
    for out in (y, q, k):
        bad = ~torch.isfinite(out).all(-1)
        assert {tuple(i) for i in bad.nonzero().tolist()} <= {(0, 2, 1), (0, 3, 0), (0, 4, 3)}
    assert torch.equal(y[..., 64:].nan_to_num(7.0), x[..., 64:].nan_to_num(7.0))
    only = ~torch.isfinite(y[0, 2, 1])
    assert only.nonzero().flatten().tolist() == [5, 37]  # the pair that holds the NaN


def _norm_case(layout, batch, seq, heads, kv, dim, dtype, seed):
    g = _gen(seed)
    q = _heads(layout, batch, seq, heads, dim, dtype, seed + 1)
    k = _heads(layout, batch, seq, kv, dim, dtype, seed + 2)
    wq = (1 + 0.2 * torch.randn(dim, generator=g, device=DEV)).to(dtype)
    wk = (1 + 0.2 * torch.randn(dim, generator=g, device=DEV)).to(dtype)
    pos = torch.randint(0, 40000, (batch, seq), generator=g, device=DEV)
    return [t.detach().requires_grad_(True) for t in (q, k, wq, wk)], pos


def _check_norm(leaves, pos, freq, dtype, interleaved, scale=1.0, eps=1e-6):
    q, k, wq, wk = leaves
    outs = helion_b200.qk_norm_rope(q, k, wq, wk, pos, freq, eps=eps, interleaved=interleaved, scale=scale)
    refs = block_oracle.qk_norm_rope(q.detach(), k.detach(), wq.detach(), wk.detach(), pos, freq, eps, interleaved, scale)
    dys = [torch.randn(t.shape, generator=_gen(9), device=DEV).to(dtype) for t in (q, k)]
    grads = torch.autograd.grad(outs, leaves, dys)
    for i, (x, w) in enumerate(((q.detach(), wq.detach()), (k.detach(), wk.detach()))):
        normed = block_oracle.head_norm(x, w, eps)
        _close(outs[i].detach(), refs[i], dtype, (2e-6 + 6e-7) * 2 * scale * _rowmax(normed))
        dx, dw, size = block_oracle.head_norm_rope_backward(dys[i], x, w, pos, freq, eps, interleaved, scale)
        gw = scale * 1.42 * _rowmax(dys[i]) * w.abs().max().double()
        rstd = (x.double().pow(2).mean(-1, keepdim=True) + eps).rsqrt()
        _close(grads[i], dx, dtype, 1e-5 * rstd * gw * (1 + _rowmax(x) * rstd))
        _close(grads[2 + i], dw, dtype, 1e-5 * size)
    return outs, grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("dim", "rotary", "interleaved"), SHAPES)
def test_qk_norm_rope_forward_and_gradients(dtype, dim, rotary, interleaved):
    leaves, pos = _norm_case("bshd", 2, 7, 5, 2, dim, dtype, dim + rotary)
    _check_norm(leaves, pos, helion_b200.rope_frequencies(rotary)[0], dtype, interleaved, scale=1.25)


@pytest.mark.parametrize("layout", ["bshd", "bhsd", "fused", "offset", "lastdim"])
@pytest.mark.parametrize(("batch", "seq", "heads", "kv"), [(1, 1, 1, 1), (4, 1, 32, 8), (2, 333, 9, 3), (1, 2000, 6, 6)])
def test_qk_norm_rope_layouts_and_lengths(layout, batch, seq, heads, kv):
    leaves, pos = _norm_case(layout, batch, seq, heads, kv, 128, torch.bfloat16, seq)
    freq, _ = helion_b200.rope_frequencies(128)
    outs, grads = _check_norm(leaves, pos, freq, torch.bfloat16, False)
    again = helion_b200.qk_norm_rope(*leaves, pos, freq)
    dys = [torch.randn(t.shape, generator=_gen(9), device=DEV).bfloat16() for t in leaves[:2]]
    for a, b in zip((*outs, *grads), (*again, *torch.autograd.grad(again, leaves, dys))):
        assert torch.equal(a, b)  # sums in a fixed order


def test_rows_of_zeros_and_tiny_values():
    leaves, pos = _norm_case("bshd", 1, 3, 2, 1, 64, torch.float32, 4)
    with torch.no_grad():
        leaves[0][0, 0] = 0.0
        leaves[0][0, 1] *= 1e-5
    _check_norm(leaves, pos, helion_b200.rope_frequencies(64)[0], torch.float32, False, eps=1e-6)


def test_gradients_for_some_inputs_only_and_broadcast_heads():
    leaves, pos = _norm_case("bshd", 2, 6, 4, 2, 64, torch.float32, 8)
    freq, _ = helion_b200.rope_frequencies(64)
    q, k, wq, wk = (t.detach() for t in leaves)
    full = helion_b200.qk_norm_rope(*leaves, pos, freq)
    dys = [torch.randn_like(t) for t in (q, k)]
    ref = torch.autograd.grad(full, leaves, dys)
    for i in range(4):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, wq, wk))]
        outs = helion_b200.qk_norm_rope(*some, pos, freq)
        assert torch.equal(torch.autograd.grad(outs, [some[i]], dys)[0], ref[i])
    # one key head shown to four query groups (stride 0), its gradient summed by autograd
    base = torch.randn(2, 6, 1, 64, generator=_gen(6), device=DEV, requires_grad=True)
    y = helion_b200.rope(base.expand(2, 6, 4, 64), pos, freq)
    dy = torch.randn(y.shape, generator=_gen(7), device=DEV)
    (got,) = torch.autograd.grad(y, base, dy)
    terms = block_oracle.rope(dy, pos, freq, inverse=True)
    _close(got, terms.sum(2, keepdim=True), torch.float32, 6e-7 * 8 * _rowmax(dy).amax(2, keepdim=True))
    # only one of the two outputs is used
    q2 = q.clone().requires_grad_(True)
    outs = helion_b200.qk_norm_rope(q2, k, wq, wk, pos, freq)
    assert torch.equal(torch.autograd.grad(outs[0], q2, dys[0])[0], ref[0])


def test_gradients_against_differences():
    """d/dt of sum(dy * f(x + t v)) at 0 by central differences of the kernel's own float32 forward at h and h / 2,
    extrapolated (the h^2 term cancels; what is left is h^4 and the forward's rounding over h)."""
    leaves, pos = _norm_case("bshd", 1, 4, 3, 2, 32, torch.float32, 12)
    freq, _ = helion_b200.rope_frequencies(32)
    dys = [torch.randn_like(t) for t in leaves[:2]]
    grads = torch.autograd.grad(helion_b200.qk_norm_rope(*leaves, pos, freq), leaves, dys)
    base = [t.detach() for t in leaves]

    def value(args):
        return float(sum((d.double() * o.double()).sum() for d, o in zip(dys, helion_b200.qk_norm_rope(*args, pos, freq))))

    for i in range(4):
        v = torch.randn(base[i].shape, generator=_gen(40 + i), device=DEV)

        def slope(h):
            up, down = ([t + s * h * v if j == i else t for j, t in enumerate(base)] for s in (1, -1))
            return (value(up) - value(down)) / (2 * h)

        h = 2.0 ** -5
        numeric = (4 * slope(h / 2) - slope(h)) / 3
        exact = float((grads[i].double() * v.double()).sum())
        size = float((grads[i].double() * v.double()).abs().sum())
        # rounding: every output is good to ~1e-6, so the difference over 2h = 1 / 32 to ~3e-5 of the magnitudes;
        # h^4 = 1e-6 times the fifth derivative of 1 / sqrt(1 + t^2), below 120
        assert abs(numeric - exact) <= 2e-4 * max(size, 1.0)


def test_second_derivative_of_rope_and_refusal_of_the_norms():
    x = torch.randn(1, 3, 2, 16, device=DEV, requires_grad=True)
    freq, _ = helion_b200.rope_frequencies(16)
    pos = torch.arange(3, device=DEV)
    y = helion_b200.rope(x, pos, freq)
    (dx,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    torch.testing.assert_close(dx, 2 * x, rtol=1e-5, atol=1e-5)  # a rotation keeps lengths
    (ddx,) = torch.autograd.grad(dx.sum(), x)
    torch.testing.assert_close(ddx, torch.full_like(x, 2.0), rtol=1e-5, atol=1e-5)
    w = torch.ones(16, device=DEV, requires_grad=True)
    q, _ = helion_b200.qk_norm_rope(x, x, w, w, pos, freq)
    (dx,) = torch.autograd.grad((q * q).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)


def test_other_streams_and_captured_graphs():
    leaves, pos = _norm_case("bshd", 2, 64, 8, 2, 128, torch.bfloat16, 20)
    freq, _ = helion_b200.rope_frequencies(128)
    dys = [torch.randn(t.shape, device=DEV).bfloat16() for t in leaves[:2]]

    def step(args):
        outs = helion_b200.qk_norm_rope(*args, pos, freq)
        return [*outs, *torch.autograd.grad(outs, args, dys)]

    expected = [t.detach().clone() for t in step(leaves)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for got, ref in zip(step(leaves), expected):
            assert torch.equal(got.detach(), ref)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    # two graphs over leaves of their own; replayed side by side they must not share scratch
    graphs, results = [], []
    for _ in range(2):
        args = [t.detach().clone().requires_grad_(True) for t in leaves]
        with torch.cuda.stream(side):
            step(args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            results.append([t.detach() for t in step(args)])
        graphs.append((g, args))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (g, _args), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for res in results:
        for got, ref in zip(res, expected):
            assert torch.equal(got, ref)
    with torch.no_grad():  # new inputs in the captured buffers
        graphs[0][1][0].mul_(0.5)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(results[1][0], expected[0])
    fresh = [t.detach().clone().requires_grad_(True) for t in graphs[0][1]]
    for got, ref in zip(results[0], step(fresh)):
        assert torch.equal(got, ref.detach())


def test_outputs_stay_inside_their_buffers():
    """Through the C ABI: strided outputs between pattern bytes; gaps and guards stay as they were."""
    L = _lib.lib()
    for dtype, code, dim, half in ((torch.bfloat16, 0, 128, 64), (torch.float32, 2, 72, 9), (torch.float16, 1, 7, 3)):
        batch, seq, heads, wide = 2, 3, 5, dim + 8
        x = torch.randn(batch, seq, heads, dim, device=DEV).to(dtype)
        out = torch.full((batch, seq, heads + 1, wide), 7.0, dtype=dtype, device=DEV)
        pos = torch.arange(seq, device=DEV)
        freq, _ = helion_b200.rope_frequencies(2 * half)
        rows = _lib.HeadRows(x.data_ptr(), x.stride()[:3], out.data_ptr(), out.stride()[:3], None, (0, 0, 0), None, None, heads)
        _lib.check(L.lce_rope(ctypes.byref(rows), batch, seq, dim, pos.data_ptr(), 1, 0, 1, freq.data_ptr(), half, 0, 1.0, 0, code,
                              torch.cuda.current_stream().cuda_stream), "lce_rope")
        torch.cuda.synchronize()
        assert torch.equal(out[:, :, :heads, :dim], helion_b200.rope(x, pos, freq))
        assert bool((out[:, :, :heads, dim:] == 7.0).all()) and bool((out[:, :, heads:] == 7.0).all())
