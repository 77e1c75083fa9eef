"""The operators of a decoder step around the LM head, as cases that can be timed and compared.

Four operators: the projection with its epilogue (``linear``), rotary positions (``rope``), the norm of every
query and key head with the rotation in the same pass (``qk_norm_rope``), and the sampler that draws tokens from
logits (``sample_logits``). ``own`` chooses between their plain form in elementary torch operations and the
framework's entry points; both take what ``prepare`` gives.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")
EPS = 1e-6


# ----------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the output projection of one decode step: 16 sequences, residual stream added in the epilogue
        dict(name="linear_decode", op="linear", m=16, k=4096, n=4096, dtype="bf16", act="none", bias=True, residual=True,
             train=False),
        # the up projection over a prompt batch, the largest product here
        dict(name="linear_prompt", op="linear", m=8192, k=4096, n=16384, dtype="bf16", act="silu", bias=False, residual=False,
             train=False),
        # the first half of a feed-forward block in training: forward, input, weight and bias gradients
        dict(name="linear_train", op="linear", m=8192, k=1024, n=4096, dtype="bf16", act="gelu", bias=True, residual=False,
             train=True),
        # a small model's projection trained in single precision, sizes that fit no tile
        dict(name="linear_train_odd", op="linear", m=777, k=520, n=1003, dtype="fp32", act="relu", bias=True, residual=True,
             train=True),
        # the keys and queries of two long prompts, all heads rotated in full, rows inside a wider projection
        dict(name="rope_prompt", op="rope", batch=2, seq=8192, heads=40, dim=128, rotary=128, dtype="bf16", interleaved=False,
             fused=True, far=0, train=True),
        # one token for each of 48 sequences far into their contexts, a part of an unusual head rotated, paired lanes
        dict(name="rope_decode", op="rope", batch=48, seq=1, heads=24, dim=80, rotary=32, dtype="fp16", interleaved=True,
             fused=False, far=1000000, train=False),
        # one training step of the attention input of a grouped-query block: all gradients
        dict(name="qknorm_train", op="qknorm", batch=4, seq=4096, heads=32, kv_heads=8, dim=128, rotary=128, dtype="bf16",
             interleaved=False, far=0, train=True),
        # one decode step of the same block for 32 sequences, straight out of the fused projection
        dict(name="qknorm_decode", op="qknorm", batch=32, seq=1, heads=32, kv_heads=8, dim=128, rotary=128, dtype="bf16",
             interleaved=False, far=30000, train=False),
        # narrow odd heads in single precision, a part rotated in pairs
        dict(name="qknorm_train_odd", op="qknorm", batch=3, seq=701, heads=5, kv_heads=1, dim=72, rotary=36, dtype="fp32",
             interleaved=True, far=5000, train=True),
        # a single conversation: the smallest draw, where the latency of the call counts
        dict(name="sample_single", op="sample", rows=1, vocab=50257, dtype="bf16", filters="top_k", masked=0.0, logprob=False),
        # a serving batch in which every request has filters of its own, a fifth of the vocabulary ruled out by a grammar
        dict(name="sample_serving", op="sample", rows=64, vocab=128256, dtype="fp32", filters="mixed", masked=0.2, logprob=True),
        # a large batch of samples for training from them, with their log-probabilities: the nucleus alone
        dict(name="sample_rollout", op="sample", rows=256, vocab=128256, dtype="bf16", filters="top_p", masked=0.0, logprob=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "rope", "qknorm", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "linear":
        train = rng.random() < 0.5
        top = 1024 if dtype == "fp32" else 4096  # single-precision models here are small
        case = dict(op=op, m=_log(rng, 1, 8192), k=_log(rng, 32, top), n=_log(rng, 32, 4 * top), dtype=dtype,
                    act=rng.choice(ACTIVATIONS), bias=rng.random() < 0.7, residual=rng.random() < 0.5, train=train)
        if rng.random() < 0.6:  # most widths are whole vectors
            case["k"], case["n"] = -(-case["k"] // 8) * 8, -(-case["n"] // 8) * 8
        case["n"] = max(1, min(case["n"], 8192 * 4096 * 16384 // ((3 if train else 1) * case["m"] * case["k"])))
        return case
    if op == "sample":
        vocab = _log(rng, 1000, 256000)
        rows = min(_log(rng, 1, 256), 256 * 128256 // vocab)
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, filters=rng.choice(["none", "top_k", "top_p", "min_p", "mixed"]),
                    masked=rng.choice([0.0, 0.0, 0.2, 0.9]), logprob=rng.random() < 0.5)
    dim = rng.choice([32, 64, 72, 80, 96, 128, 192, 256])
    rotary = rng.choice([dim, dim, dim // 2, 2 * (dim // 8)])
    train = rng.random() < 0.5
    seq = 1 if rng.random() < 0.4 else _log(rng, 2, 8192)
    heads = rng.choice([1, 3, 8, 16, 32, 40])
    batch = _log(rng, 1, 128)
    budget = 2 * 8192 * 40 * 128 // (2 if dtype == "fp32" else 1)
    batch = max(1, min(batch, budget // (seq * heads * dim * 2)))
    seq = max(1, min(seq, budget // (batch * heads * dim * 2)))
    case = dict(op=op, batch=batch, seq=seq, heads=heads, dim=dim, rotary=rotary, dtype=dtype, interleaved=rng.random() < 0.5,
                far=rng.choice([0, 5000, 100000, 1000000]), train=train)
    if op == "rope":
        case["fused"] = rng.random() < 0.5
    else:
        case["kv_heads"] = rng.choice([h for h in (1, 2, 4, 8) if h <= heads])
    return case


def _sizes(case):
    elt = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "linear":
        return elt, case["m"] * case["k"], case["n"] * case["k"], case["m"] * case["n"]
    return elt, case["batch"] * case["seq"], case["heads"] + case.get("kv_heads", 0), case["dim"]


def work(case):
    if case["op"] == "linear":
        elt, x, w, y = _sizes(case)
        n = case["n"] if case["bias"] else 0
        moved = x + w + n + y + (y if case["residual"] else 0)  # x, W, bias and residual in, y out
        flops = 2 * case["m"] * case["k"] * case["n"]
        if case["train"]:
            moved += y + x + w + n  # dy in; dX, dW, dbias out
            flops *= 3
        return {"bytes": elt * moved, "flops": flops}
    if case["op"] == "sample":
        elt = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * elt + 4 + 20 + (12 if case["logprob"] else 8)), "flops": 4 * case["rows"] * case["vocab"]}
    elt, tokens, heads, dim = _sizes(case)
    elements = tokens * heads * dim
    small = tokens * 8 + case["rotary"] // 2 * 8
    if case["op"] == "rope":  # forward, and backward over the gradient
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * elements * elt + small, "flops": passes * 3 * elements}
    moved = (2 + 2 if case["train"] else 2) * elements * elt  # x in, out; with gradients dy in, dx out
    return {"bytes": moved + (4 if case["train"] else 2) * dim * elt + small, "flops": (18 if case["train"] else 7) * elements}


# ----------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)

    st = dict(case)
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        st["x"] = normal(m, k).requires_grad_(case["train"])
        st["w"] = normal(n, k, std=k ** -0.5).requires_grad_(case["train"])
        st["b"] = normal(n, std=0.1).requires_grad_(case["train"]) if case["bias"] else None
        st["r"] = normal(m, n) if case["residual"] else None
        st["dy"] = normal(m, n) if case["train"] else None
        return st
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn(rows, vocab, generator=g, device=dev) * 2.0  # a model's logits: a broad bulk and a few favourites
        favoured = torch.randint(0, vocab, (rows, 24), generator=g, device=dev)
        logits.scatter_(1, favoured, 6.0 + 3.0 * torch.randn(rows, 24, generator=g, device=dev))
        if case["masked"]:
            logits.masked_fill_(torch.rand(rows, vocab, generator=g, device=dev) < case["masked"], float("-inf"))
        st["logits"] = logits.to(dtype)
        st["u"] = torch.rand(rows, generator=g, device=dev)

        def spread(low, high):
            return low + (high - low) * torch.rand(rows, generator=g, device=dev)

        filters = case["filters"]
        st["temperature"] = spread(0.6, 1.3)
        top_k = torch.randint(1, 200, (rows,), generator=g, device=dev)
        top_p, min_p = spread(0.5, 0.99), spread(0.01, 0.2)
        if filters == "mixed":  # requests differ in which of the filters they set; some are greedy
            on = torch.rand(3, rows, generator=g, device=dev) < 0.6
            st["temperature"] = torch.where(torch.rand(rows, generator=g, device=dev) < 0.1, 0.0, st["temperature"])
            st["top_k"] = torch.where(on[0], top_k, 0)
            st["top_p"] = torch.where(on[1], top_p, 1.0)
            st["min_p"] = torch.where(on[2], min_p, 0.0)
        else:
            st["top_k"] = top_k if filters == "top_k" else torch.zeros_like(top_k)
            st["top_p"] = top_p if filters == "top_p" else torch.ones_like(top_p)
            st["min_p"] = min_p if filters == "min_p" else torch.zeros_like(min_p)
        return st
    batch, seq, heads, dim, rotary = (case[i] for i in ("batch", "seq", "heads", "dim", "rotary"))
    if case["far"]:  # every sequence somewhere of its own in a long context
        start = torch.randint(0, case["far"], (batch, 1), generator=g, device=dev)
    else:
        start = torch.zeros((batch, 1), dtype=torch.int64, device=dev)
    st["positions"] = start + torch.arange(seq, device=dev)
    st["frequencies"] = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=dev) / rotary)
    if case["op"] == "rope":
        if case["fused"]:  # the heads are a slice of a wider projection's output
            x = normal(batch, seq, heads + 8, dim)[:, :, :heads]
        else:
            x = normal(batch, seq, heads, dim)
        st["x"] = x.requires_grad_(case["train"])
        st["dy"] = normal(batch, seq, heads, dim) if case["train"] else None
        return st
    kv = case["kv_heads"]
    qkv = normal(batch, seq, heads + 2 * kv, dim)
    st["q"] = qkv[:, :, :heads].requires_grad_(case["train"])
    st["k"] = qkv[:, :, heads:heads + kv].requires_grad_(case["train"])
    st["wq"] = (1.0 + normal(dim, std=0.1)).requires_grad_(case["train"])
    st["wk"] = (1.0 + normal(dim, std=0.1)).requires_grad_(case["train"])
    if case["train"]:
        st["dq"], st["dk"] = normal(batch, seq, heads, dim), normal(batch, seq, kv, dim)
    return st


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------
def run(st):
    if own:
        return _own(st)
    with torch.no_grad():
        return {"linear": _plain_linear, "rope": _plain_rope, "qknorm": _plain_qknorm, "sample": _plain_sample}[st["op"]](st)


def _own(st):
    import helion_b200

    if st["op"] == "linear":
        act = None if st["act"] == "none" else st["act"]
        y = helion_b200.linear(st["x"], st["w"], st["b"], activation=act, residual=st["r"])
        if not st["train"]:
            return [y]
        leaves = [t for t in (st["x"], st["w"], st["b"]) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, st["dy"])]
    if st["op"] == "sample":
        drawn = helion_b200.sample_logits(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                                          top_p=st["top_p"], min_p=st["min_p"], return_logprob=st["logprob"])
        return list(drawn) if st["logprob"] else [drawn]
    if st["op"] == "rope":
        y = helion_b200.rope(st["x"], st["positions"], st["frequencies"], interleaved=st["interleaved"])
        return [y.detach(), *torch.autograd.grad(y, [st["x"]], st["dy"])] if st["train"] else [y]
    q, k = helion_b200.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["positions"], st["frequencies"], eps=EPS,
                                    interleaved=st["interleaved"])
    if not st["train"]:
        return [q, k]
    grads = torch.autograd.grad([q, k], [st["q"], st["k"], st["wq"], st["wk"]], [st["dq"], st["dk"]])
    return [q.detach(), k.detach(), *grads]


# ---- plain forms: 32 bits throughout, one rounding at the end ---------------------------------------------------
def _plain_act(z, act):
    """act(z) and its derivative."""
    if act == "relu":
        return torch.clamp_min(z, 0.0), (z > 0).float()
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _plain_linear(st):
    dtype = st["x"].dtype
    x, w = st["x"].float(), st["w"].float()
    z = x @ w.t()
    if st["b"] is not None:
        z = z + st["b"].float()
    y, slope = _plain_act(z, st["act"])
    if st["r"] is not None:
        y = y + st["r"].float()
    if not st["train"]:
        return [y.to(dtype)]
    dz = st["dy"].float() * slope
    grads = [dz @ w, dz.t() @ x] + ([dz.sum(0)] if st["b"] is not None else [])
    return [t.to(dtype) for t in [y, *grads]]


def _plain_angles(st):
    angle = st["positions"].double()[..., None, None] * st["frequencies"]  # far positions lose their angle in 32 bits
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_rotate(x, cos, sin, rotary, interleaved):
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., rotary:]], dim=-1)


def _plain_rope(st):
    dtype = st["x"].dtype
    cos, sin = _plain_angles(st)
    y = _plain_rotate(st["x"].float(), cos, sin, st["rotary"], st["interleaved"]).to(dtype)
    if not st["train"]:
        return [y]
    return [y, _plain_rotate(st["dy"].float(), cos, -sin, st["rotary"], st["interleaved"]).to(dtype)]


def _plain_qknorm(st):
    dtype = st["q"].dtype
    cos, sin = _plain_angles(st)

    def normed(x, w):
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        return x * rstd, rstd, _plain_rotate(x * rstd * w, cos, sin, st["rotary"], st["interleaved"])

    def gradients(dy, unit, rstd, w):
        dn = _plain_rotate(dy, cos, -sin, st["rotary"], st["interleaved"])
        dw = (dn * unit).flatten(0, -2).double().sum(0)  # tens of thousands of rows: a long sum
        dn = dn * w
        return rstd * (dn - unit * (dn * unit).mean(-1, keepdim=True)), dw

    wq, wk = st["wq"].float(), st["wk"].float()
    uq, rq, q = normed(st["q"].float(), wq)
    uk, rk, k = normed(st["k"].float(), wk)
    if not st["train"]:
        return [q.to(dtype), k.to(dtype)]
    gq, gwq = gradients(st["dq"].float(), uq, rq, wq)
    gk, gwk = gradients(st["dk"].float(), uk, rk, wk)
    return [t.to(dtype) for t in (q, k, gq, gk, gwq, gwk)]


def _plain_sample(st):
    logits = torch.nan_to_num(st["logits"].double(), nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    vocab = logits.shape[1]
    values, order = torch.sort(logits, dim=1, descending=True, stable=True)  # of equal values the lower index first
    top = values[:, :1]
    temperature = st["temperature"].double()[:, None]
    greedy = temperature <= 0
    # 64 bits: the draw compares sums of up to the whole vocabulary with a bound that may lie next to one of them
    weights = torch.exp((values - top) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(vocab, device=logits.device)
    limit = torch.where(st["top_k"] > 0, st["top_k"], vocab)[:, None]
    limit = torch.where(greedy, 1, limit)
    weights = torch.where(rank < limit, weights, 0.0)
    sums = torch.cumsum(weights, dim=1)
    ahead = sums - weights
    top_p = st["top_p"].double()[:, None]
    keep = (weights > 0) & ((ahead <= top_p * sums[:, -1:]) | (top_p >= 1.0)) & (weights >= st["min_p"].double()[:, None])
    kept = torch.zeros_like(weights).scatter_(1, order, torch.where(keep, weights, 0.0))  # back into the vocabulary's order
    sums = torch.cumsum(kept, dim=1)
    bound = st["u"].double()[:, None] * sums[:, -1:]
    token = ((sums <= bound) | (kept == 0)).long().cummin(dim=1).values.sum(1)
    if not st["logprob"]:
        return [token]
    return [token, torch.log(kept.gather(1, token[:, None])[:, 0] / sums[:, -1]).float()]


# ----------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------
def _exact_sample(st):
    tokens, logprobs = [], []
    for row in range(st["rows"]):
        logits, u = st["logits"][row].double(), st["u"][row].double()
        t, k, p, m = (float(st[i][row]) for i in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            tokens.append(torch.nonzero(logits == logits.max())[0, 0])
            logprobs.append(torch.zeros((), dtype=torch.float64, device=logits.device))
            continue
        prob = torch.softmax(logits / t, 0)
        ranked = torch.argsort(logits, descending=True, stable=True)[:int(k) if k > 0 else None]
        share = prob[ranked] / prob[ranked].sum()
        inside = (share.cumsum(0) - share <= p) if p < 1 else torch.ones_like(share, dtype=torch.bool)
        inside &= (share >= m * share[0]) & (share > 0)
        index = torch.sort(ranked[inside]).values
        line = prob[index].cumsum(0)
        pick = torch.searchsorted(line, u * line[-1], right=True).clamp_max(len(index) - 1)
        tokens.append(index[pick])
        logprobs.append(torch.log(prob[index[pick]] / line[-1]))
    return [torch.stack(tokens), torch.stack(logprobs)] if st["logprob"] else [torch.stack(tokens)]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    if case["op"] == "linear":
        wide = {i: st[i].detach().double().requires_grad_(case["train"]) for i in ("x", "w", "b", "r") if st[i] is not None}
        z = torch.nn.functional.linear(wide["x"], wide["w"], wide.get("b"))
        y = {"none": lambda t: t, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t),
             "gelu": lambda t: t * torch.special.ndtr(t),
             "gelu_tanh": lambda t: t * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3))}[case["act"]](z)
        y = y + wide["r"] if "r" in wide else y
        if not case["train"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, [wide[i] for i in ("x", "w", "b") if i in wide], st["dy"].double())]
    half = case["rotary"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       st["positions"][:, :, None, None].double() * st["frequencies"])

    def rotated(x):
        pairs = x[..., :case["rotary"]]
        if case["interleaved"]:
            pairs = pairs.unflatten(-1, (half, 2))
        else:
            pairs = pairs.unflatten(-1, (2, half)).transpose(-1, -2)
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        return torch.cat([pairs.flatten(-2), x[..., case["rotary"]:]], -1)

    if case["op"] == "rope":
        x = st["x"].detach().double().requires_grad_(case["train"])
        y = rotated(x)
        return [y.detach(), *torch.autograd.grad(y, [x], st["dy"].double())] if case["train"] else [y]
    q, k, wq, wk = (st[i].detach().double().requires_grad_(case["train"]) for i in ("q", "k", "wq", "wk"))
    outs = [rotated(t * (t.pow(2).mean(-1, keepdim=True) + EPS).pow(-0.5) * w) for t, w in ((q, wq), (k, wk))]
    if not case["train"]:
        return outs
    return [t.detach() for t in outs] + list(torch.autograd.grad(outs, [q, k, wq, wk], [st["dq"].double(), st["dk"].double()]))
