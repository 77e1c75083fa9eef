"""linear against its float64 definition: activations, types, odd and strided shapes, gradients, capture. GPU only.

Tolerances, from arithmetic. u = 2^-24. A sum of K products in 32 bits is off by at most K u S, S the sum of their
magnitudes (products of 16-bit values are exact). The activations are Lipschitz with 1.13, their derivatives with 0.8, and
computed to 4e-6 of their magnitude. One rounding of the result: eps / 2. In the backward pass act' is taken at z
rounded to the input type (0.8 |z| eps / 2 in the slope) and dz is rounded as an operand (|dz| eps / 2); both then pass
through the products, whose sums obey the first rule. At a z within its own error of 0 relu's slope may be either."""

from __future__ import annotations

import pytest
import torch

import helion_b200
from helion_b200 import _lib
from oracle import block_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inside(got, ref, bound, what):
    assert got.shape == ref.shape, what
    over = ((got.double() - ref).abs() - bound).max() if ref.numel() else torch.zeros(())
    assert over <= 0, f"{what}: off by {float(over):.3e} more than the bound"


def _half(dtype):
    info = torch.finfo(dtype)
    return info.eps / 2 * (1 + info.eps), info.tiny * info.eps


def _check(x, w, b, r, act, dy=None, y=None):
    """Forward, and with dy the gradients, against float64; returns what was computed."""
    dtype = x.dtype
    half, tiny = _half(dtype)
    m, k = x.shape
    n = w.shape[0]
    ref, z = block_oracle.linear(x.detach(), w.detach(), None if b is None else b.detach(), act,
                                 None if r is None else r.detach())
    xa, wa = x.detach().double().abs(), w.detach().double().abs()
    z_err = (k + 1) * U * (xa @ wa.t() + (0 if b is None else b.detach().double().abs()))
    y = helion_b200.linear(x, w, b, activation=act, residual=r)
    assert y.dtype == dtype
    size = ref.abs() + (0 if r is None else 2 * r.detach().double().abs())
    _inside(y.detach(), ref, half * ref.abs() + tiny + 1.13 * z_err + 4e-6 * size, "y")
    if dy is None:
        return [y]
    leaves = [t for t in (x, w, b, r) if t is not None and t.requires_grad]
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy)))
    dx, dw, db, dz = block_oracle.linear_backward(dy, x.detach(), w.detach(), None if b is None else b.detach(), act)
    dya = dy.double().abs()
    if act == "relu":
        slope_err = (z.abs() <= z_err).double()
    elif act is None:
        slope_err = torch.zeros_like(z)
    else:
        slope_err = 0.8 * (z.abs() * half + tiny + z_err) + 4e-6 * (1 + z.abs())
    unrounded = dya * slope_err + 2 * U * dz.abs()
    dz_err = unrounded + (0 if act is None else half * dz.abs() + tiny)
    dza = dz.abs() + dz_err
    _inside(grads[id(x)], dx, half * dx.abs() + tiny + dz_err @ wa + n * U * (dza @ wa), "dx")
    _inside(grads[id(w)], dw, half * dw.abs() + tiny + dz_err.t() @ xa + m * U * (dza.t() @ xa), "dw")
    if b is not None:
        _inside(grads[id(b)], db, half * db.abs() + tiny + unrounded.sum(0) + m * U * dza.sum(0), "dbias")
    if r is not None and r.requires_grad:
        assert torch.equal(grads[id(r)], dy)
    return [y, *grads.values()]


def _case(m, k, n, dtype, bias=True, residual=True, grad=True, seed=0):
    g = _gen(seed + m + 3 * k + 7 * n)

    def make(*shape, std=1.0):
        return (std * torch.randn(*shape, generator=g, device=DEV)).to(dtype).requires_grad_(grad)

    return (make(m, k), make(n, k, std=k ** -0.5), make(n, std=0.3) if bias else None, make(m, n) if residual else None,
            make(m, n).detach())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize(("bias", "residual"), [(True, True), (False, False), (True, False), (False, True)])
def test_every_epilogue(dtype, act, bias, residual):
    x, w, b, r, dy = _case(70, 136, 200, dtype, bias, residual)
    _check(x, w, b, r, act, dy)


SHAPES = [(1, 8, 8), (1, 1, 1), (1, 4096, 256), (3, 7, 5), (16, 4096, 520), (128, 64, 1024), (129, 100, 257), (300, 72, 1000),
          (257, 513, 33), (2, 2048, 2056), (1000, 31, 9), (2049, 40, 264), (64, 8192, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("m", "k", "n"), SHAPES)
def test_odd_and_skewed_shapes(dtype, m, k, n):
    x, w, b, r, dy = _case(m, k, n, dtype)
    first = _check(x, w, b, r, "silu", dy)
    second = _check(x, w, b, r, "silu", dy)
    for a, c in zip(first, second):
        assert torch.equal(a, c)  # sums in a fixed order
    with torch.no_grad():
        assert torch.equal(helion_b200.linear(x, w, b, activation="silu", residual=r), first[0])


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 64, 65, 127])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_decode_batches(dtype, m):
    """A handful of tokens: every batch size in turn, a contraction that is and one that is not whole vectors."""
    for k, n in ((1024, 776), (1003, 130)):
        x, w, b, r, _ = _case(m, k, n, dtype, grad=False)
        _check(x, w, b, r, "gelu")
        _check(x, w, None, None, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_pitches_and_leading_dimensions(dtype):
    g = _gen(4)
    base = torch.randn(6, 50, 3 * 64, generator=g, device=DEV).to(dtype)
    w_wide = torch.randn(96, 80, generator=g, device=DEV).to(dtype)
    r_wide = torch.randn(6, 50, 100, generator=g, device=DEV).to(dtype)
    b = torch.randn(192, generator=g, device=DEV).to(dtype)[::2]
    for lo in (0, 64, 3):  # aligned and unaligned slices of a fused projection
        x, w, r = base[:, :, lo:lo + 64], w_wide[:, lo % 16:lo % 16 + 64], r_wide[:, :, lo % 5:lo % 5 + 96]
        y = helion_b200.linear(x, w, b, activation="relu", residual=r)
        assert y.shape == (6, 50, 96)
        plain = helion_b200.linear(x.contiguous(), w.contiguous(), b.contiguous(), activation="relu", residual=r.contiguous())
        assert torch.equal(y, plain)
        _check(x.reshape(300, 64), w, b, r.reshape(300, 96), "relu")
    # transposed, expanded and one-dimensional inputs
    xt = torch.randn(64, 30, generator=g, device=DEV).to(dtype).t()
    w = w_wide[:, :64]
    assert torch.equal(helion_b200.linear(xt, w), helion_b200.linear(xt.contiguous(), w))
    wt = torch.randn(64, 40, generator=g, device=DEV).to(dtype).t()
    assert torch.equal(helion_b200.linear(base[..., :64], wt), helion_b200.linear(base[..., :64], wt.contiguous()))
    one = base[0, 0, :64]
    assert torch.equal(helion_b200.linear(one, w, residual=r_wide[0, 0, :96]),
                       helion_b200.linear(one[None], w, residual=r_wide[:1, 0, :96])[0])
    assert torch.equal(helion_b200.linear(one.expand(5, 64), w), helion_b200.linear(one.repeat(5, 1), w))


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_batches(dtype):
    x = torch.randn(0, 16, device=DEV).to(dtype).requires_grad_(True)
    w = torch.randn(24, 16, device=DEV).to(dtype).requires_grad_(True)
    b = torch.randn(24, device=DEV).to(dtype).requires_grad_(True)
    y = helion_b200.linear(x, w, b, activation="gelu")
    assert y.shape == (0, 24)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == (0, 16) and bool((dw == 0).all()) and bool((db == 0).all())
    assert helion_b200.linear(torch.randn(2, 0, 16, device=DEV).to(dtype), w.detach()).shape == (2, 0, 24)


def test_gradients_for_some_inputs_only_and_expanded_gradients():
    x, w, b, r, dy = _case(90, 64, 48, torch.bfloat16)
    ref = torch.autograd.grad(helion_b200.linear(x, w, b, activation="gelu", residual=r), (x, w, b, r), dy)
    for i in range(4):
        some = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate((x, w, b, r))]
        y = helion_b200.linear(some[0], some[1], some[2], activation="gelu", residual=some[3])
        assert torch.equal(torch.autograd.grad(y, some[i], dy)[0], ref[i])
    y = helion_b200.linear(x, w, b, activation="silu")
    ones = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    y = helion_b200.linear(x, w, b, activation="silu")
    for a, c in zip(ones, torch.autograd.grad(y.sum(), (x, w, b))):  # the gradient arrives with strides of 0
        assert torch.equal(a, c)
    # x serves as its own residual: both gradients arrive
    sq = torch.randn(40, 48, device=DEV).bfloat16().requires_grad_(True)
    ww = torch.randn(48, 48, device=DEV).bfloat16()
    y = helion_b200.linear(sq, ww, residual=sq)
    d = torch.randn_like(y)
    (got,) = torch.autograd.grad(y, sq, d)
    assert torch.equal(got, helion_b200.linear(d, ww.t()) + d)
    y = helion_b200.linear(x, w, b, activation="gelu")
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), w)


@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh", "silu"])
def test_gradients_against_differences(act):
    """Central differences of the kernel's own float32 forward at h and h / 2, extrapolated."""
    x, w, b, r, dy = _case(9, 12, 10, torch.float32)
    leaves = [x, w, b, r]
    grads = torch.autograd.grad(helion_b200.linear(x, w, b, activation=act, residual=r), leaves, dy)
    base = [t.detach() for t in leaves]
    for i in range(4):
        v = torch.randn(base[i].shape, generator=_gen(60 + i), device=DEV)

        def value(s):
            a = [t + s * v if j == i else t for j, t in enumerate(base)]
            return float((helion_b200.linear(a[0], a[1], a[2], activation=act, residual=a[3]).double() * dy.double()).sum())

        def slope(h):
            return (value(h) - value(-h)) / (2 * h)

        h = 2.0 ** -5
        numeric = (4 * slope(h / 2) - slope(h)) / 3
        exact = float((grads[i].double() * v.double()).sum())
        size = float((grads[i].double().abs() * v.double().abs()).sum()) + 90.0
        # rounding: ~1e-6 of 90 outputs over 2 h = 1 / 32; the h^4 term: 1e-6 times a fifth derivative of order 10
        assert abs(numeric - exact) <= 2e-4 * size


def test_extreme_values():
    x = torch.tensor([[1e4], [-1e4], [88.0], [-88.0], [0.0], [300.0], [-300.0], [1e-8]], device=DEV)
    for dtype in DTYPES:
        w = torch.ones(8, 1, device=DEV, dtype=dtype).requires_grad_(True)
        for act in ACTS:
            xd = x.to(dtype).requires_grad_(True)
            y = helion_b200.linear(xd, w, activation=act)
            ref = block_oracle.activation(xd.detach(), act)
            half, tiny = _half(dtype)
            _inside(y.detach(), ref[0].expand(8, 8), half * ref[0].abs() + 4e-6 * ref[0].abs() + tiny, f"{act} {dtype}")
            (dx,) = torch.autograd.grad(y, xd, torch.ones_like(y))
            slope_err = 4e-6 + half * (0.8 * xd.detach().double().abs() * (act not in (None, "relu")) + ref[1].abs())
            slope_err = torch.where(xd.detach().abs() > 80, 1e-6, slope_err)
            _inside(dx, 8 * ref[1], half * 8 * ref[1].abs() + 8 * slope_err, f"{act} {dtype} slope")
    inf = torch.tensor([[float("inf")], [3e38], [-3e38]], device=DEV)
    for dtype in (torch.bfloat16, torch.float32):
        for act in ACTS:
            y = helion_b200.linear(inf.to(dtype), torch.ones(8, 1, device=DEV, dtype=dtype), activation=act)
            assert bool((y[0] == float("inf")).all()) and bool((y[1] > 2.9e38).all())
            assert act is None or bool((y[2] == 0).all())
    for act in ACTS:  # a NaN stays in its row
        xb = torch.randn(40, 64, device=DEV).bfloat16()
        xb[7, 3] = float("nan")
        y = helion_b200.linear(xb, torch.randn(72, 64, device=DEV).bfloat16(), activation=act)
        assert bool(torch.isnan(y[7]).all()) and bool(torch.isfinite(y[torch.arange(40, device=DEV) != 7]).all())


def test_other_streams_and_captured_graphs():
    x, w, b, r, dy = _case(16, 4096, 512, torch.bfloat16)  # a split contraction: the call uses scratch

    def step(args):
        y = helion_b200.linear(args[0], args[1], args[2], activation="gelu", residual=args[3])
        return [y.detach(), *torch.autograd.grad(y, args, dy)]

    expected = [t.clone() for t in step([x, w, b, r])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for got, ref in zip(step([x, w, b, r]), expected):
            assert torch.equal(got, ref)
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):
        args = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]
        with torch.cuda.stream(side):
            step(args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            results.append(step(args))
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


@pytest.mark.parametrize(("m", "k", "n", "ldo", "dtype"), [(70, 100, 190, 200, torch.bfloat16), (1, 64, 7, 9, torch.float16),
                                                           (300, 65, 129, 131, torch.bfloat16), (33, 20, 50, 64, torch.float32),
                                                           (5, 4096, 40, 48, torch.bfloat16)])
def test_outputs_stay_inside_their_buffers(m, k, n, ldo, dtype):
    L = _lib.lib()
    code = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}[dtype]
    x, w, b, r, dy = _case(m, k, n, dtype, grad=False)
    out = torch.full((m + 2, ldo), 7.0, dtype=dtype, device=DEV)
    saved = m * ((n + 7) // 8 * 8)
    pre = torch.full((saved + 64,), 7.0, dtype=dtype, device=DEV)
    need = L.lce_linear_forward_workspace_bytes(x.data_ptr(), k, w.data_ptr(), k, m, n, k, code, 0)
    ws = torch.full((need + 512,), 90, dtype=torch.uint8, device=DEV)
    s = torch.cuda.current_stream().cuda_stream
    _lib.check(L.lce_linear_forward(x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), r.data_ptr(), n, out.data_ptr(), ldo,
                                    pre.data_ptr(), m, n, k, 4, code, ws.data_ptr(), need, 0, s), "lce_linear_forward")
    torch.cuda.synchronize()
    assert torch.equal(out[:m, :n], helion_b200.linear(x, w, b, activation="silu", residual=r))
    assert bool((out[m:] == 7.0).all()) and bool((out[:, n:] == 7.0).all()) and bool((pre[saved:] == 7.0).all())
    assert bool((ws[need:] == 90).all())
    grads = [torch.full((size + 64,), 7.0, dtype=dtype, device=DEV) for size in (m * k, n * k, n)]
    args = (dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k)
    need = L.lce_linear_backward_workspace_bytes(*args, m, n, k, 4, code, 0)
    ws = torch.full((need + 512,), 90, dtype=torch.uint8, device=DEV)
    _lib.check(L.lce_linear_backward(*args, pre.data_ptr(), *(t.data_ptr() for t in grads), m, n, k, 4, code, ws.data_ptr(), need,
                                     0, s), "lce_linear_backward")
    torch.cuda.synchronize()
    for t, size in zip(grads, (m * k, n * k, n)):
        assert bool((t[size:] == 7.0).all())
    assert bool((ws[need:] == 90).all()) and _lib.device_status() == 0


def test_forced_kernel_families(monkeypatch):
    x, w, b, r, dy = _case(150, 96, 264, torch.bfloat16)
    for force in ("simt", "tc", "tc1"):
        monkeypatch.setenv("HELION_B200_FORCE", force)
        _check(x, w, b, r, "gelu_tanh", dy)
    x, w, b, r, dy = _case(30, 33, 40, torch.float32)
    monkeypatch.setenv("HELION_B200_FORCE", "tc")  # fp32 has one family
    _check(x, w, b, r, "gelu", dy)
