"""sample_logits against its definition in float64: filters alone and together, ties, masks, values that are not
finite, strides, batch sizes, capture. GPU only.

Tokens have to be equal. Both sides form weights and sums in 64 bits; where the definition puts a draw ON a boundary
between two tokens (periodic weights and a uniform of 1/2 do), the rounding of a 64-bit sum decides, and the oracle
names both. Boundaries between sums that are exact - of equal weights - are tested by value. Log-probabilities are
rounded to float32 once."""

from __future__ import annotations

import pytest
import torch

import helion_b200
from helion_b200 import _lib
from oracle import block_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
INF = float("inf")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(rows, vocab, dtype, seed, masked=0.0):
    g = _gen(seed)
    l = 2.0 * torch.randn(rows, vocab, generator=g, device=DEV)
    l.scatter_(1, torch.randint(0, vocab, (rows, 8), generator=g, device=DEV), 6 + 3 * torch.randn(rows, 8, generator=g, device=DEV))
    if masked:
        l.masked_fill_(torch.rand(rows, vocab, generator=g, device=DEV) < masked, -INF)
    return l.to(dtype)


def _f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


def _check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Each parameter a scalar or a list of one per row."""
    rows = logits.shape[0]

    def given(v, dtype):
        return torch.tensor(v, dtype=dtype, device=DEV) if isinstance(v, list) else v

    token, logprob = helion_b200.sample_logits(
        logits, u, temperature=given(temperature, torch.float32), top_k=given(top_k, torch.int32),
        top_p=given(top_p, torch.float32), min_p=given(min_p, torch.float32), return_logprob=True)
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32 and token.shape == logprob.shape == (rows,)

    def row(v, i):
        return v[i] if isinstance(v, list) else v

    for i in range(rows):
        want = block_oracle.sample(logits[i], float(u[i]), _f32(row(temperature, i)), row(top_k, i), _f32(row(top_p, i)),
                                   _f32(row(min_p, i)))
        assert int(token[i]) in want, f"row {i}: {int(token[i])}, not {want}"
        got, lp = float(logprob[i]), want[int(token[i])]
        assert got == lp or abs(got - lp) <= 2.0 ** -23 * abs(lp) + 1e-9, f"row {i}: logprob {got}, not {lp}"
    return token, logprob


FILTERS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_k=1000), dict(top_p=0.1), dict(top_p=0.9),
           dict(top_p=0.999), dict(min_p=0.05), dict(min_p=1.0), dict(temperature=1.3, top_k=200, top_p=0.8, min_p=0.02),
           dict(temperature=0.3, top_k=5, top_p=0.5), dict(temperature=0), dict(temperature=50.0, top_p=0.5),
           dict(temperature=0.01, top_p=0.99), dict(top_k=64, min_p=0.3), dict(top_k=3000, top_p=0.97)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("filters", FILTERS, ids=lambda f: "-".join(f"{k}{v}" for k, v in f.items()) or "none")
def test_filters(dtype, filters):
    for vocab in (1000, 5003):
        logits = _logits(7, vocab, dtype, vocab)
        _check(logits, torch.rand(7, generator=_gen(3), device=DEV), **filters)


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 31, 33, 255, 1023, 1024, 1025, 4097, 32000, 50257, 128256, 256000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_vocabulary_sizes(dtype, vocab):
    rows = 3
    logits = _logits(rows, vocab, dtype, vocab) if vocab > 8 else torch.randn(rows, vocab, generator=_gen(1), device=DEV).to(dtype)
    u = torch.rand(rows, generator=_gen(vocab), device=DEV)
    _check(logits, u)
    _check(logits, u, temperature=0.9, top_k=max(1, vocab // 3), top_p=0.95, min_p=0.001)
    _check(logits, u, top_p=0.7)


def test_parameters_of_every_row():
    rows = 24
    logits = _logits(rows, 3001, torch.float32, 5, masked=0.2)
    u = torch.rand(rows, generator=_gen(8), device=DEV)
    temperature = [0.0, 1.0, 0.5, -1.0, 2.0, 0.7] * 4
    top_k = [0, 1, 50, -3, 5000, 3001] * 4
    top_p = [1.0, 0.5, 0.9, 2.0, 0.0, -1.0, 0.95, 0.2] * 3
    min_p = [0.0, 0.1, -0.5, 1.0, 0.02, 3.0, 0.0, 0.001] * 3
    a, _ = _check(logits, u, temperature, top_k, top_p, min_p)
    b = helion_b200.sample_logits(logits, u, temperature=torch.tensor(temperature, device=DEV),
                                  top_k=torch.tensor(top_k, device=DEV), top_p=torch.tensor(top_p, device=DEV),
                                  min_p=torch.tensor(min_p, device=DEV))
    assert torch.equal(a, b)  # int64 top_k, no log-probabilities
    for i in range(0, rows, 5):  # a row does not depend on its neighbours, nor on how its parameters arrive
        if temperature[i] >= 0 and top_k[i] >= 0 and 0 < top_p[i] <= 1 and 0 <= min_p[i] <= 1:
            one = helion_b200.sample_logits(logits[i], u[i], temperature=temperature[i], top_k=top_k[i], top_p=top_p[i],
                                            min_p=min_p[i])
            assert one.shape == () and int(one) == int(a[i])


def test_ties_go_to_the_lower_index():
    vocab = 600
    flat = torch.zeros(1, vocab, device=DEV)
    for u, want in ((0.0, 0), (0.5, 300), (0.25, 150), (1 - 2.0 ** -24, 599), (0.125, 75)):
        _check(flat, torch.tensor([u], device=DEV))
        assert int(helion_b200.sample_logits(flat[0], torch.tensor(u, device=DEV))) == want  # sums of ones are exact
    for dtype in DTYPES:
        steps = (torch.arange(vocab, device=DEV) % 3).to(dtype)[None].contiguous()  # 200 each of 0, 1, 2
        for u in (0.0, 0.3, 0.5, 0.75, 0.99):
            uu = torch.tensor([u], device=DEV)
            for k in (1, 7, 199, 200, 201, 399, 400, 401, 599):
                _check(steps, uu, top_k=k)
            for p in (0.001, 0.25, 0.5, 0.6, 0.665, 0.9, 0.9999):
                _check(steps, uu, top_p=p)
                _check(steps, uu, top_p=p, top_k=250)
    # the boundary itself: of 8 equal tokens, a top_p of 1/2 keeps those with at most 4 ahead, five
    eight = torch.full((1, 8), 3.0, device=DEV)
    assert int(helion_b200.sample_logits(eight, torch.tensor([1 - 2.0 ** -24], device=DEV), top_p=0.5)) == 4
    zeros = torch.tensor([[-0.0, 0.0, -0.0, 0.0]], device=DEV)  # the two zeros are one logit
    for dtype in DTYPES:
        assert int(helion_b200.sample_logits(zeros.to(dtype), torch.tensor([0.9], device=DEV), top_k=1)) == 0
        assert int(helion_b200.sample_logits(zeros.to(dtype), torch.tensor([0.9], device=DEV), top_k=2)) == 1


def test_masked_rows_and_values_that_are_not_finite():
    for dtype in DTYPES:
        low = torch.finfo(dtype).min
        l = _logits(10, 777, dtype, 6)
        l[0] = -INF
        l[1] = float("nan")
        l[2, :] = -INF
        l[2, 500] = 1.0
        l[3, 100] = float("nan")
        l[4, 5], l[4, 600] = INF, INF
        l[5] = low
        l[6, 3:] = low
        l[7, ::2] = -INF
        l[8] = torch.finfo(dtype).max
        l[9] = -INF
        l[9, :3] = low
        for u in (0.0, 0.4, 0.99):
            uu = torch.full((10,), u, device=DEV)
            for f in (dict(), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.5), dict(temperature=0), dict(top_k=600, top_p=0.999),
                      dict(temperature=1e-30), dict(temperature=1e30, top_p=0.3)):
                token, lp = _check(l, uu, **f)
                assert int(token[0]) == -1 and float(lp[0]) == -INF and int(token[2]) == 500
    odd = torch.tensor([0.5, -1.0, 2.0, INF, -INF, float("nan")], device=DEV)  # uniforms out of their range are clamped
    flat = torch.zeros(6, 10, device=DEV)
    assert helion_b200.sample_logits(flat, odd).tolist() == [5, 0, 9, 9, 0, 0]
    weird = helion_b200.sample_logits(flat, odd, temperature=torch.tensor([INF, float("nan"), 1.0, 1.0, 1.0, 1.0], device=DEV),
                                      top_p=torch.tensor([float("nan")] * 6, device=DEV), min_p=torch.tensor([float("nan")] * 6, device=DEV))
    assert weird.tolist() == [5, 0, 9, 9, 0, 0]


@pytest.mark.parametrize("rows", [1, 2, 37, 150, 300, 1000])
def test_batches(rows):
    logits = _logits(rows, 2050, torch.bfloat16, rows)
    u = torch.rand(rows, generator=_gen(rows), device=DEV)
    token, _ = _check(logits, u, temperature=1.1, top_k=300, top_p=0.9)
    again = helion_b200.sample_logits(logits, u, temperature=1.1, top_k=300, top_p=0.9)
    assert torch.equal(token, again)


@pytest.mark.parametrize("layout", ["rows", "view"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_batches_with_rows_of_every_kind(dtype, layout):
    """A batch that large bf16 calls take in another form, each row with filters of its own: ordinary rows, masked ones,
    ties, zeros of both signs, rows of values that have no bin of their own (tiny, huge, infinite), nothing kept, NaN."""
    rows, vocab = 72, 32771
    wide = _logits(rows, vocab + 13, dtype, 31)
    logits = wide[:, 5:5 + vocab] if layout == "view" else wide[:, :vocab].contiguous()
    g = _gen(32)
    largest = torch.finfo(dtype).max
    for i in range(8):  # every kind meets eight of the filters
        at = 9 * i
        logits[at + 1].masked_fill_(torch.rand(vocab, generator=g, device=DEV) < 0.9, -INF)
        logits[at + 2, ::7] = 3e-7 if dtype == torch.float16 else 1e-12
        logits[at + 3, 5::1001] = largest / 2
        logits[at + 4, 17 * (i + 1)::9001] = INF
        logits[at + 5] = torch.randint(-4, 5, (vocab,), generator=g, device=DEV).to(dtype)
        logits[at + 6] = torch.where(torch.rand(vocab, generator=g, device=DEV) < 0.5, 0.0, -0.0).to(dtype)
        logits[at + 7, ::3] = float("nan")
        logits[at + 8] = -INF if i % 2 else -2.75
    u = torch.rand(rows, generator=_gen(33), device=DEV)
    u[3], u[4] = 0.0, 1.0
    params = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    lists = {name: [FILTERS[(5 * i + i // 9) % len(FILTERS)].get(name, off) for i in range(rows)] for name, off in params.items()}
    first = _check(logits, u, **lists)
    second = _check(logits.clone(), u, **lists)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])


@pytest.mark.parametrize("filters", FILTERS)
def test_large_batches_of_one_kind(filters):
    logits = _logits(64, 31253, torch.bfloat16, 41)
    _check(logits, torch.rand(64, generator=_gen(42), device=DEV), **filters)


def test_peaked_flat_and_wide_spread_logits():
    vocab = 70000
    u = torch.tensor([0.0, 0.2, 0.7, 0.999999], device=DEV)
    ramp = torch.linspace(-80, 0, vocab, device=DEV)
    cases = [torch.zeros(vocab, device=DEV), ramp, ramp.flip(0), ramp * 1e-4, 1e4 * ramp,
             torch.where(torch.arange(vocab, device=DEV) == 69999, 30.0, 0.0), torch.full((vocab,), -INF, device=DEV).index_fill_(0, torch.tensor([5, 60000], device=DEV), 2.0)]
    for c in cases:
        l = c.expand(4, vocab).contiguous()
        for f in (dict(), dict(top_p=0.5), dict(top_p=0.99), dict(top_k=30000), dict(top_k=30000, top_p=0.8), dict(min_p=0.01),
                  dict(temperature=0.05, top_p=0.9)):
            _check(l, u, **f)
        _check(l.bfloat16(), u, top_p=0.9)


def test_views_and_leading_dimensions():
    g = _gen(9)
    wide = torch.randn(4, 3, 1200, generator=g, device=DEV)
    u = torch.rand(4, 3, generator=g, device=DEV)
    for view in (wide, wide[..., 5:1000], wide[..., ::2], wide.transpose(0, 1).contiguous().transpose(0, 1), wide[:, :, :1].expand(4, 3, 50)):
        got, lp = helion_b200.sample_logits(view, u, top_p=0.9, return_logprob=True)
        flat = helion_b200.sample_logits(view.reshape(12, -1).contiguous(), u.reshape(12), top_p=0.9)
        assert got.shape == lp.shape == (4, 3) and torch.equal(got.reshape(12), flat)
    ut = torch.rand(3, 4, generator=g, device=DEV).t()
    assert torch.equal(helion_b200.sample_logits(wide, ut), helion_b200.sample_logits(wide, ut.contiguous()))
    assert helion_b200.sample_logits(wide[:0], u[:0]).shape == (0, 3)
    sliced = wide[:, 1, 7:900]  # rows a wider pitch apart, off 16-byte boundaries
    _check(sliced, u[:, 0].contiguous(), top_k=50, top_p=0.9)


def test_a_large_row_count_of_draws_follows_the_distribution():
    """40000 draws from 6 tokens: counts within 6 standard deviations of the binomial."""
    n = 40000
    l = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5, -INF], device=DEV).expand(n, 6).contiguous()
    token = helion_b200.sample_logits(l, torch.rand(n, generator=_gen(77), device=DEV))
    p = torch.softmax(l[0].double(), 0)
    for j in range(6):
        c, e = float((token == j).sum()), float(p[j]) * n
        assert abs(c - e) <= 6 * (e * (1 - float(p[j]))) ** 0.5


def test_streams_and_captured_graphs():
    logits = _logits(9, 20000, torch.bfloat16, 4)
    u = torch.rand(9, generator=_gen(4), device=DEV)
    kw = dict(temperature=torch.full((9,), 0.9, device=DEV), top_k=400, top_p=0.95)
    expected = helion_b200.sample_logits(logits, u, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(helion_b200.sample_logits(logits, u, **kw), expected)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        l, uu = logits.clone(), u.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = helion_b200.sample_logits(l, uu, return_logprob=True, **kw)
        graphs.append((g, l, uu, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (g, *_rest), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _g, _l, _u, out in graphs:
        assert torch.equal(out[0], expected)
    g, l, uu, out = graphs[0]
    l.copy_(_logits(9, 20000, torch.bfloat16, 14))
    uu.copy_(torch.rand(9, generator=_gen(15), device=DEV))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], helion_b200.sample_logits(l, uu, **kw))


def test_outputs_stay_inside_their_buffers():
    L = _lib.lib()
    rows, vocab, ld = 5, 1001, 1010
    logits = torch.randn(rows, ld, device=DEV).bfloat16()
    logits[:, vocab:] = float("inf")  # what lies between the rows is not read
    u = torch.rand(rows, device=DEV)
    token = torch.full((rows + 8,), -7, dtype=torch.int64, device=DEV)
    logprob = torch.full((rows + 8,), 7.0, device=DEV)
    need = L.lce_sample_logits_workspace_bytes(rows, vocab, 0)
    ws = torch.full((need + 512,), 90, dtype=torch.uint8, device=DEV)
    _lib.check(L.lce_sample_logits(logits.data_ptr(), ld, rows, vocab, 0, u.data_ptr(), None, 0.8, None, 0, 30, None, 0.9, None,
                                   0.01, token.data_ptr(), logprob.data_ptr(), ws.data_ptr(), need,
                                   torch.cuda.current_stream().cuda_stream), "lce_sample_logits")
    torch.cuda.synchronize()
    assert torch.equal(token[:rows], helion_b200.sample_logits(logits[:, :vocab], u, temperature=0.8, top_k=30, top_p=0.9, min_p=0.01))
    assert bool((token[rows:] == -7).all()) and bool((logprob[rows:] == 7.0).all()) and bool((ws[need:] == 90).all())


def test_agrees_with_the_sampling_head_on_its_candidates():
    """Where sample_head's candidates suffice, the two describe the same distribution."""
    from helion_b200 import decode_ops

    g = _gen(30)
    hidden = torch.randn(6, 128, generator=g, device=DEV)
    weight = torch.randn(900, 128, generator=g, device=DEV) * 0.3
    idx, probs = decode_ops.sampling_distribution(hidden, weight, temperature=0.8, top_k=20, top_p=0.7)
    logits = helion_b200.matmul(hidden, weight.t())
    for u in (0.05, 0.35, 0.65, 0.95):
        token, lp = helion_b200.sample_logits(logits, torch.full((6,), u, device=DEV), temperature=0.8, top_k=20, top_p=0.7,
                                              return_logprob=True)
        for i in range(6):
            at = (idx[i] == token[i]).nonzero()[0, 0]
            assert abs(float(lp[i].exp()) - float(probs[i, at])) <= 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("equal", [1, 2, 3, 511, 1023, 1024, 1025])
def test_lists_of_candidates(dtype, equal):
    """A top_k whose candidates are few enough to be listed, up to and past the list's 1024: `equal` logits share the
    k-th value, so the lower indices are kept; some lie above, some far below."""
    vocab = 6007
    g = _gen(90 + equal)
    order = torch.randperm(vocab, generator=g, device=DEV)
    row = torch.full((vocab,), -3.0, device=DEV)
    row[order[:equal]] = 2.0
    above = [] if equal >= 1023 else [2.5, 3.0, 3.0, 4.0]
    for i, v in enumerate(above):
        row[order[equal + i]] = v
    row[order[equal + 10:equal + 500]] = -INF
    ks = sorted({1, 2, max(1, equal // 2), equal, equal + len(above), equal + len(above) + 1})
    u = torch.linspace(0, 1, len(ks), device=DEV)
    logits = row.to(dtype).expand(len(ks), vocab).contiguous()
    _check(logits, u, top_k=ks)
    _check(logits, u, temperature=0.6, top_k=ks, top_p=[0.3 + 0.1 * (i % 6) for i in range(len(ks))], min_p=0.1)
