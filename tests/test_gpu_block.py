"""The operators of a decoder block together, as a model uses them: a decode step down to the drawn token, eager and as
a captured graph, and a training step down to the loss of the fused head. GPU only.

Forward links are compared, each from the inputs that it had, with their float64 definitions under the bounds that
arithmetic gives: K 2^-24 of the magnitudes of a sum of K products, 2e-6 for a normalised element, 6e-7 for a rotation,
half a step for each rounding. A backward link must give the bits that the operator gives alone for the same incoming
gradient (its own tests hold those against the formulas), so nothing of a neighbour, a workspace or a stream may leak
in. The whole gradient in 32 bits is held against float64: about 20 links, each good to 5e-6 of its magnitudes
(74 x 2^-24 for sums of up to 64 terms), with orthonormal weights, so that a link amplifies an error by less
than 10: 1e-3 of the largest element."""

from __future__ import annotations

import math
import threading

import pytest
import torch

import helion_b200
from oracle import block_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HIDDEN, HEADS, KV, DIM, FFN, VOCAB = 256, 4, 2, 64, 512, 1003


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inside(got, ref, bound, what):
    half = torch.finfo(got.dtype)
    bound = bound + half.eps / 2 * (1 + half.eps) * ref.abs() + half.tiny * half.eps
    over = float(((got.double() - ref).abs() - bound).max())
    assert over <= 0, f"{what}: off by {over:.3e} more than the bound"


def _weights(dtype, seed, hidden=HIDDEN, heads=HEADS, kv=KV, dim=DIM, ffn=FFN):
    g = _gen(seed)

    def rand(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device=DEV)).to(dtype)

    return {
        "norm1": 1 + rand(hidden, scale=0.1), "norm2": 1 + rand(hidden, scale=0.1),
        "qkv": rand((heads + 2 * kv) * dim, hidden, scale=hidden ** -0.5), "qkv_bias": rand((heads + 2 * kv) * dim, scale=0.1),
        "qn": 1 + rand(dim, scale=0.1), "kn": 1 + rand(dim, scale=0.1), "out": rand(hidden, heads * dim, scale=(heads * dim) ** -0.5),
        "up": rand(ffn, hidden, scale=hidden ** -0.5), "up_bias": rand(ffn, scale=0.1), "down": rand(hidden, ffn, scale=ffn ** -0.5),
    }


def _split(qkv, heads=HEADS, kv=KV, dim=DIM):
    """[..., (heads + 2 kv) dim] -> q, k, v as strided views of it."""
    t = qkv.unflatten(-1, (heads + 2 * kv, dim))
    return t[..., :heads, :], t[..., heads:heads + kv, :], t[..., heads + kv:, :]


def _attend(q, keys, values, allowed):
    """Plain attention. q [B, Q, heads, D], keys and values [B, L, kv, D], allowed [B, Q, L]."""
    groups = q.shape[2] // keys.shape[2]
    keys, values = (t[:, :, :, None].expand(-1, -1, -1, groups, -1).flatten(2, 3).to(q.dtype) for t in (keys, values))
    scores = torch.einsum("bqhd,blhd->bhql", q, keys) / math.sqrt(q.shape[-1])
    p = scores.masked_fill(~allowed[:, None], -math.inf).softmax(-1)
    return torch.einsum("bhql,blhd->bqhd", p, values)


def _decode_step(w, head, x, position, freq, keys, values, u):
    """One token of every sequence; returns every link's result by name. The cache rows at `position` are written."""
    batch = x.shape[0]
    at = {"n1": helion_b200.rmsnorm(x, w["norm1"])}
    at["qkv"] = helion_b200.linear(at["n1"], w["qkv"], w["qkv_bias"])
    q, k, v = _split(at["qkv"])
    at["q"], at["k"] = helion_b200.qk_norm_rope(q, k, w["qn"], w["kn"], position, freq)
    rows = torch.arange(batch, device=DEV)
    keys.index_put_((rows, position), at["k"])
    values.index_put_((rows, position), v)
    allowed = torch.arange(keys.shape[1], device=DEV) <= position[:, None]
    at["attn"] = _attend(at["q"][:, None].float(), keys, values, allowed[:, None])[:, 0].to(x.dtype).flatten(1)
    at["x1"] = helion_b200.linear(at["attn"], w["out"], residual=x)
    at["n2"] = helion_b200.rmsnorm(at["x1"], w["norm2"])
    at["up"] = helion_b200.linear(at["n2"], w["up"], w["up_bias"], activation="silu")
    at["x2"] = helion_b200.linear(at["up"], w["down"], residual=at["x1"])
    at["logits"] = helion_b200.linear(at["x2"], head)
    at["token"], at["logprob"] = helion_b200.sample_logits(at["logits"], u, temperature=0.8, top_k=50, top_p=0.9, min_p=0.01,
                                                           return_logprob=True)
    return at


def _check_linear(got, x, weight, bias=None, act=None, residual=None, what=""):
    ref, _ = block_oracle.linear(x, weight, bias, act, residual)
    size = x.double().abs() @ weight.double().abs().t() + (0 if bias is None else bias.double().abs())
    rest = ref.abs() + (0 if residual is None else 2 * residual.double().abs())
    _inside(got, ref, 1.13 * (x.shape[-1] + 1) * U * size + 4e-6 * rest, what)


def _decode_inputs(batch, length, dtype, seed):
    g = _gen(seed)
    x = torch.randn(batch, HIDDEN, generator=g, device=DEV).to(dtype)
    position = torch.randint(0, length, (batch,), generator=g, device=DEV)
    position[0] = 0  # a sequence that has no history
    keys, values = (torch.randn(batch, length, KV, DIM, generator=g, device=DEV).to(dtype) for _ in range(2))
    head = (torch.randn(VOCAB, HIDDEN, generator=g, device=DEV) * 3 * HIDDEN ** -0.5).to(dtype)
    u = torch.rand(batch, generator=g, device=DEV)
    return head, x, position, keys, values, u


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("batch", [1, 3, 33, 70])
@torch.no_grad()
def test_decode_step(batch, dtype):
    w = _weights(dtype, 1)
    head, x, position, keys, values, u = _decode_inputs(batch, 48, dtype, 2 + batch)
    freq, scale = helion_b200.rope_frequencies(DIM, theta=10000.0)
    assert scale == 1.0
    at = _decode_step(w, head, x, position, freq, keys, values, u)
    _check_linear(at["qkv"], at["n1"], w["qkv"], w["qkv_bias"], what="qkv")
    q, k, v = _split(at["qkv"])
    for got, ref, t, weight in zip((at["q"], at["k"]),
                                   block_oracle.qk_norm_rope(q, k, w["qn"], w["kn"], position, freq), (q, k), (w["qn"], w["kn"])):
        normed = block_oracle.head_norm(t, weight, 1e-6)
        _inside(got, ref, 2 * 2.6e-6 * normed.abs().amax(-1, keepdim=True), "qk_norm_rope")
    rows = torch.arange(batch, device=DEV)
    assert torch.equal(keys[rows, position], at["k"]) and torch.equal(values[rows, position], v)
    _check_linear(at["x1"], at["attn"], w["out"], residual=x, what="x1")
    _check_linear(at["up"], at["n2"], w["up"], w["up_bias"], "silu", what="up")
    _check_linear(at["x2"], at["up"], w["down"], residual=at["x1"], what="x2")
    _check_linear(at["logits"], at["x2"], head, what="logits")
    f32 = [float(torch.tensor(f, dtype=torch.float32)) for f in (0.8, 0.9, 0.01)]
    for i in range(batch):
        want = block_oracle.sample(at["logits"][i], float(u[i]), f32[0], 50, f32[1], f32[2])
        token = int(at["token"][i])
        assert token in want and abs(float(at["logprob"][i]) - want[token]) <= 2.0 ** -23 * abs(want[token]) + 1e-9


@pytest.mark.parametrize("batch", [1, 5])
@torch.no_grad()
def test_two_captured_decode_loops(batch):
    """Two graphs of the step, each with buffers of its own, replayed on two streams at once for several tokens: the token
    drawn is fed back on the device. Both must give what the eager loop gives."""
    dtype, steps = torch.bfloat16, 6
    w = _weights(dtype, 3)
    freq, _ = helion_b200.rope_frequencies(DIM, theta=10000.0)
    embed = torch.randn(VOCAB, HIDDEN, generator=_gen(4), device=DEV).to(dtype)
    draws = [torch.rand(steps, batch, generator=_gen(s), device=DEV) for s in (5, 6)]

    def fresh(seed):
        head, x, _, keys, values, u = _decode_inputs(batch, steps + 2, dtype, seed)
        return dict(head=head, x=x, position=torch.zeros(batch, dtype=torch.int64, device=DEV), keys=keys, values=values, u=u)

    def step(s):
        at = _decode_step(w, s["head"], s["x"], s["position"], freq, s["keys"], s["values"], s["u"])
        s["x"].copy_(embed[at["token"]])
        s["position"].add_(1)
        return at["token"], at["logprob"]

    expected = []
    for i in range(2):
        state = fresh(10 + i)
        run = []
        for n in range(steps):
            state["u"].copy_(draws[i][n])
            run.append([t.clone() for t in step(state)])
        expected.append(run)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    loops = []
    for i in range(2):
        state, start = fresh(10 + i), fresh(10 + i)
        with torch.cuda.stream(side):
            step(state)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            result = step(state)
        for name, t in state.items():
            t.copy_(start[name])
        loops.append((graph, state, result))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in loops]
    got = [[], []]
    for n in range(steps):
        for i, (graph, state, result) in enumerate(loops):
            with torch.cuda.stream(streams[i]):
                state["u"].copy_(draws[i][n])
                graph.replay()
                got[i].append([t.clone() for t in result])
    torch.cuda.synchronize()
    for i in range(2):
        for n in range(steps):
            assert all(torch.equal(a, b) for a, b in zip(got[i][n], expected[i][n])), (i, n)


def _train_step(ops, w, head, x, target, positions, freq, heads, kv, dim, watch):
    """A causal block and the loss; `watch(name, tensor)` sees each link's result. ops: rmsnorm, linear, qk_norm_rope, loss."""
    batch, seq, _ = x.shape
    n1 = watch("n1", ops["rmsnorm"](x, w["norm1"]))
    qkv = watch("qkv", ops["linear"](n1, w["qkv"], w["qkv_bias"], None, None))
    q, k, v = _split(qkv, heads, kv, dim)
    q, k = ops["qk_norm_rope"](q, k, w["qn"], w["kn"], positions, freq)
    q, k = watch("q", q), watch("k", k)
    allowed = torch.ones(seq, seq, dtype=torch.bool, device=x.device).tril().expand(batch, seq, seq)
    attn = watch("attn", _attend(q, k, v, allowed).flatten(2))
    x1 = watch("x1", ops["linear"](attn, w["out"], None, None, x))
    n2 = watch("n2", ops["rmsnorm"](x1, w["norm2"]))
    up = watch("up", ops["linear"](n2, w["up"], w["up_bias"], "gelu_tanh", None))
    x2 = watch("x2", ops["linear"](up, w["down"], None, None, x1))
    return ops["loss"](x2, head, target)


OPS = {
    "rmsnorm": helion_b200.rmsnorm,
    "linear": lambda x, w, b, act, r: helion_b200.linear(x, w, b, activation=act, residual=r),
    "qk_norm_rope": helion_b200.qk_norm_rope,
    "loss": lambda x, head, target: helion_b200.linear_cross_entropy(x, head, target),
}
PLAIN = {  # float64, differentiated by torch
    "rmsnorm": lambda x, w: x * (x.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w,
    "linear": lambda x, w, b, act, r: block_oracle.linear(x, w, b, act, r)[0],
    "qk_norm_rope": block_oracle.qk_norm_rope,
    "loss": lambda x, head, target: torch.nn.functional.cross_entropy((x @ head.t()).flatten(0, 1), target.flatten()),
}


def _train_inputs(dtype, batch, seq, hidden, heads, kv, dim, ffn, seed):
    w = _weights(dtype, seed, hidden, heads, kv, dim, ffn)
    g = _gen(seed + 1)
    x = torch.randn(batch, seq, hidden, generator=g, device=DEV).to(dtype)
    head = (torch.randn(VOCAB, hidden, generator=g, device=DEV) * hidden ** -0.5).to(dtype)
    target = torch.randint(0, VOCAB, (batch, seq), generator=g, device=DEV)
    positions = torch.arange(seq, device=DEV).expand(batch, seq) + torch.arange(batch, device=DEV)[:, None] * 7
    return w, head, x, target, positions


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(("batch", "seq"), [(1, 1), (2, 37), (3, 64)])
def test_training_step_links(batch, seq, dtype):
    """Every operator's gradients inside the step are, bit for bit, those that it gives alone."""
    w, head, x, target, positions = _train_inputs(dtype, batch, seq, HIDDEN, HEADS, KV, DIM, FFN, 20)
    freq, _ = helion_b200.rope_frequencies(DIM, theta=10000.0)
    leaves = {**w, "head": head, "x": x}
    for t in leaves.values():
        t.requires_grad_(True)
    at = {}

    def watch(name, t):
        t.retain_grad()
        at[name] = t
        return t

    def run():
        at.clear()
        for t in leaves.values():
            t.grad = None
        loss = _train_step(OPS, w, head, x, target, positions, freq, HEADS, KV, DIM, watch)
        loss.backward()
        return loss.detach()

    loss = run()
    assert torch.isfinite(loss)
    first = {k: t.grad.clone() for k, t in {**leaves, **at}.items()}  # "qkv" and "up" are the activations

    def alone(f, inputs, dys):
        inputs = [t.detach().clone().requires_grad_(True) for t in inputs]
        out = f(*inputs)
        outs = out if isinstance(out, tuple) else (out,)
        return torch.autograd.grad(outs, inputs, dys)

    q, k, _ = _split(at["qkv"].detach())
    dq, dk, dwq, dwk = alone(lambda *a: helion_b200.qk_norm_rope(*a, positions, freq), (q, k, w["qn"], w["kn"]),
                             (first["q"], first["k"]))
    assert torch.equal(dwq, first["qn"]) and torch.equal(dwk, first["kn"])
    got_q, got_k, _ = _split(first["qkv"])
    assert torch.equal(dq, got_q) and torch.equal(dk, got_k)
    dx, dw, db = alone(lambda a, b, c: helion_b200.linear(a, b, c), (at["n1"], w["qkv"], w["qkv_bias"]), (first["qkv"],))
    assert torch.equal(dx, first["n1"]) and torch.equal(dw, w["qkv"].grad)
    assert torch.equal(db, first["qkv_bias"])
    dx, dw = alone(helion_b200.linear, (at["attn"], w["out"]), (first["x1"],))
    assert torch.equal(dx, first["attn"]) and torch.equal(dw, first["out"])
    dx, dw, db = alone(lambda a, b, c: helion_b200.linear(a, b, c, activation="gelu_tanh"),
                       (at["n2"], w["up"], w["up_bias"]), (first["up"],))
    assert torch.equal(dx, first["n2"]) and torch.equal(dw, w["up"].grad) and torch.equal(db, first["up_bias"])
    dx, dw = alone(helion_b200.linear, (at["up"], w["down"]), (first["x2"],))
    assert torch.equal(dx, first["up"]) and torch.equal(dw, first["down"])
    weights = {k: t.grad.clone() for k, t in leaves.items()}
    assert torch.equal(run(), loss)
    for k, t in leaves.items():
        assert torch.equal(t.grad, weights[k]), k


def test_training_step_gradients():
    """The whole step in 32 bits against float64: every leaf's gradient, and one direction against differences."""
    hidden, heads, kv, dim, ffn = 64, 4, 2, 16, 64
    w, head, x, target, positions = _train_inputs(torch.float32, 2, 19, hidden, heads, kv, dim, ffn, 30)
    for name in ("out", "up", "down"):  # orthonormal
        w[name] = torch.linalg.qr(w[name].double())[0].float().contiguous()
    w["qkv"] = torch.linalg.qr(w["qkv"].double())[0].float().contiguous()
    freq, _ = helion_b200.rope_frequencies(dim, theta=10000.0)

    def leaves_of(dtype):
        return {k: t.detach().to(dtype).requires_grad_(True) for k, t in {**w, "head": head, "x": x}.items()}

    def loss_of(ops, t):
        return _train_step(ops, t, t["head"], t["x"], target, positions, freq, heads, kv, dim, lambda _n, v: v)

    ours, plain = leaves_of(torch.float32), leaves_of(torch.float64)
    loss, ref = loss_of(OPS, ours), loss_of(PLAIN, plain)
    assert abs(float(loss.detach()) - float(ref.detach())) <= 1e-4
    got = dict(zip(ours, torch.autograd.grad(loss, list(ours.values()))))
    want = dict(zip(plain, torch.autograd.grad(ref, list(plain.values()))))
    for name in got:
        worst = float((got[name].double() - want[name]).abs().max())
        assert worst <= 1e-3 * float(want[name].abs().max()), f"{name}: {worst:.3e}"
    # along the gradient itself the loss grows by its squared norm; a central difference of the float64 loss is good to
    # h^2 / 6 of the third derivative, which stays below 1e-2 of the slope for steps of 1e-4
    with torch.no_grad():
        norm = math.sqrt(sum(float(g.double().pow(2).sum()) for g in got.values()))
        ends = [float(loss_of(PLAIN, {k: t + sign * 1e-4 * got[k].double() / norm for k, t in plain.items()})) for sign in (1, -1)]
    assert abs((ends[0] - ends[1]) / 2e-4 - norm) <= 1e-2 * norm


def test_training_step_captured():
    """The step with its backward pass as a graph: replays follow new inputs as a graph captured on those does, to the
    bit. The loss head of so few tokens takes its separate tail launches while a stream is captured, whose sums of a
    row's 4 partial sums have another order than the eager call's: a few dozen roundings of numbers up to 8, 2e-5."""
    dtype = torch.bfloat16
    w, head, x, target, positions = _train_inputs(dtype, 2, 32, HIDDEN, HEADS, KV, DIM, FFN, 40)
    freq, _ = helion_b200.rope_frequencies(DIM, theta=10000.0)
    names = [*w, "head", "x"]

    def grads(t):
        loss = _train_step(OPS, t, t["head"], t["x"], target, positions, freq, HEADS, KV, DIM, lambda _n, v: v)
        return [loss.detach(), *torch.autograd.grad(loss, [t[n] for n in names])]

    def leaves(x_value):
        return {k: t.detach().clone().requires_grad_(True) for k, t in {**w, "head": head, "x": x_value}.items()}

    side = torch.cuda.Stream()

    def captured(t):  # leaves of the graph's own: no eager graph of them lives
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            grads(t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            result = grads(t)
        return graph, result

    expected = []
    for value in (x, x.flip(1)):
        graph, result = captured(leaves(value))
        graph.replay()
        torch.cuda.synchronize()
        expected.append([t.clone() for t in result])
        assert abs(float(result[0]) - float(grads(leaves(value))[0])) <= 2e-5
    assert not torch.equal(expected[0][-1], expected[1][-1])
    mine = leaves(x)
    graph, result = captured(mine)
    for value, want in zip((x, x.flip(1), x), (expected[0], expected[1], expected[0])):
        with torch.no_grad():
            mine["x"].copy_(value)
        graph.replay()
        torch.cuda.synchronize()
        for name, a, b in zip(["loss", *names], result, want):
            assert torch.equal(a, b), name


def test_threads_that_share_a_stream():
    """Calls of several launches from four threads at once, all on the default stream: their launches interleave there,
    so each thread's scratch must be its own."""
    dtype, rounds = torch.bfloat16, 40
    freq, _ = helion_b200.rope_frequencies(DIM, theta=10000.0)

    def make(seed):
        g = _gen(seed)
        tensors = [torch.randn(s, generator=g, device=DEV).to(dtype).requires_grad_(True)
                   for s in ((40, 2048), (96, 2048), (200, HEADS, DIM), (200, KV, DIM), (DIM,), (DIM,))]
        return tensors, torch.randn(40, 96, generator=g, device=DEV).to(dtype), torch.randint(0, 999, (200,), generator=g, device=DEV)

    def work(tensors, dy, pos):
        x, w, q, k, qw, kw = tensors
        y = helion_b200.linear(x, w, activation="silu")
        heads = helion_b200.qk_norm_rope(q, k, qw, kw, pos, freq)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dy), *torch.autograd.grad(heads, (q, k, qw, kw), heads)]

    cases = [make(50 + i) for i in range(4)]
    expected = [work(*c) for c in cases]
    wrong, ready = [], threading.Barrier(len(cases))

    def run(i):
        try:
            ready.wait(60)
            for _ in range(rounds):
                got = work(*cases[i])
                if not all(torch.equal(a, b) for a, b in zip(got, expected[i])):
                    wrong.append(f"thread {i}: other results")
                    return
        except Exception as e:  # a thread's exception would be lost
            wrong.append(f"thread {i}: {e!r}")

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not any(t.is_alive() for t in threads) and not wrong, wrong


@pytest.mark.parametrize("how", ["checkpoint", "on_cpu"])
def test_saved_tensors_that_move(how):
    """Activation checkpointing and saved tensors kept on the host: the backward pass sees other tensors than the forward
    saved, at other addresses, and must give the same bits."""
    from torch.utils.checkpoint import checkpoint

    dtype = torch.bfloat16
    w, _, x, _, positions = _train_inputs(dtype, 2, 24, HIDDEN, HEADS, KV, DIM, FFN, 60)
    freq, _ = helion_b200.rope_frequencies(DIM, theta=10000.0)
    leaves = [t.detach().requires_grad_(True) for t in (x, w["qkv"], w["qkv_bias"], w["qn"], w["kn"])]

    def block(x, weight, bias, qn, kn):
        heads = helion_b200.linear(x, weight, bias, activation="gelu").unflatten(-1, (HEADS + 2 * KV, DIM))
        q, k = helion_b200.qk_norm_rope(heads[:, :, :HEADS], heads[:, :, HEADS:HEADS + KV], qn, kn, positions.clone(), freq.clone())
        return q, k, helion_b200.rope(heads[:, :, HEADS + KV:], positions.clone(), freq.clone())

    plain = block(*leaves)
    dys = [torch.randn(t.shape, generator=_gen(61), device=DEV).to(dtype) for t in plain]
    expected = torch.autograd.grad(plain, leaves, dys)
    if how == "checkpoint":
        outs = checkpoint(block, *leaves, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu():
            outs = block(*leaves)
    noise = [torch.randn(1 << 16, device=DEV) for _ in range(8)]  # takes the addresses that were freed
    got = torch.autograd.grad(outs, leaves, dys)
    assert len(noise) == 8
    for a, b in zip([*outs, *got], [*plain, *expected]):
        assert torch.equal(a, b)


def test_inference_mode():
    w = _weights(torch.bfloat16, 70)
    head, x, position, keys, values, u = _decode_inputs(4, 16, torch.bfloat16, 71)
    freq, _ = helion_b200.rope_frequencies(DIM, theta=10000.0)
    results = []
    for guard in (torch.no_grad, torch.inference_mode):
        with guard():
            at = _decode_step(w, head, x.clone(), position, freq, keys.clone(), values.clone(), u)
            results.append([at["token"].clone(), at["logprob"].clone(), at["logits"].clone()])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_offsets_beyond_32_bits():
    """Tensors of more than 2^31 elements: the last rows, whose offsets pass 32 bits, are those of a small call."""
    g = _gen(80)
    m, k, n = 70001, 64, 32768
    x = torch.randn(m, k, generator=g, device=DEV).bfloat16().requires_grad_(True)
    w = (torch.randn(n, k, generator=g, device=DEV) / 8).bfloat16().requires_grad_(True)
    b = torch.randn(n, generator=g, device=DEV).bfloat16().requires_grad_(True)
    y = helion_b200.linear(x, w, b, activation="relu")
    assert y.numel() > 2 ** 31
    dy = torch.empty_like(y).normal_(generator=g)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    rows, cols = slice(m - 300, m), [0, 1, 777, n - 1]
    tail = helion_b200.linear(x.detach()[rows].clone(), w.detach(), b.detach(), activation="relu")
    assert torch.equal(y.detach()[rows], tail)
    xd, wd, bd = (t.detach().double() for t in (x, w, b))

    def slopes(xs, ws, bs, dys):  # dz, and how far it may be off where z is within its rounding of 0
        z = xs @ ws.t() + bs
        unsure = z.abs() <= (k + 1) * U * (xs.abs() @ ws.abs().t() + bs.abs())
        return dys.double() * (z > 0), dys.double().abs() * unsure

    dz, off = slopes(xd[rows], wd, bd, dy[rows])
    _inside(dx[rows], dz @ wd, (n + 1) * U * (dz.abs() @ wd.abs()) + off @ wd.abs(), "dx")
    dz, off = slopes(xd, wd[cols], bd[cols], dy[:, cols])
    _inside(dw[cols], dz.t() @ xd, (m + 1) * U * (dz.abs().t() @ xd.abs()) + off.t() @ xd.abs(), "dw")
    _inside(db[cols], dz.sum(0), (m + 1) * U * dz.abs().sum(0) + off.sum(0), "dbias")
    del y, dy, dx, dw, db, dz, off, tail

    heads = torch.empty(1, 66000, 256, 128, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    assert heads.numel() > 2 ** 31
    positions = torch.arange(66000, device=DEV)[None]
    freq, _ = helion_b200.rope_frequencies(128)
    out = helion_b200.rope(heads, positions, freq)
    part = slice(65900, 66000)
    assert torch.equal(out[:, part], helion_b200.rope(heads[:, part].clone(), positions[:, part], freq))
    weight = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    q, kk = helion_b200.qk_norm_rope(heads, heads[:, :, :2], weight, weight, positions, freq)
    small = helion_b200.qk_norm_rope(heads[:, part].clone(), heads[:, part, :2].clone(), weight, weight, positions[:, part], freq)
    assert torch.equal(q[:, part], small[0]) and torch.equal(kk[:, part], small[1])
    del out, q, kk, small

    for dtype in (torch.bfloat16, torch.float16):
        logits = heads.view(16896, -1).to(dtype)  # 128000 tokens
        u = torch.rand(16896, generator=g, device=DEV)
        token, logprob = helion_b200.sample_logits(logits, u, top_p=0.9, return_logprob=True)
        last, last_logprob = helion_b200.sample_logits(logits[-70:].clone(), u[-70:], top_p=0.9, return_logprob=True)
        assert torch.equal(token[-70:], last) and torch.equal(logprob[-70:], last_logprob)
