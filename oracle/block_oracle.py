"""Plain float64 definitions of the operators of a decoder block around the head: rotary positions, query / key
norms, projections with their epilogue and the sampler. What the tests compare the kernels with; any device."""

from __future__ import annotations

import math

import torch


def rope(x, positions, frequencies, interleaved=False, scale=1.0, inverse=False):
    """float64 rotation of the first 2 * len(frequencies) elements of the last dimension of x [..., heads, dim]."""
    x = x.double()
    angle = positions.double()[..., None, None] * frequencies.double()
    if inverse:
        angle = -angle
    cos, sin = torch.cos(angle) * scale, torch.sin(angle) * scale
    half = frequencies.shape[0]
    out = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., b] * cos + x[..., a] * sin
    return out


def head_norm(x, weight, eps):
    x = x.double()
    return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double()


def qk_norm_rope(q, k, q_weight, k_weight, positions, frequencies, eps=1e-6, interleaved=False, scale=1.0):
    return tuple(rope(head_norm(t, w, eps), positions, frequencies, interleaved, scale)
                 for t, w in ((q, q_weight), (k, k_weight)))


def head_norm_rope_backward(dy, x, weight, positions, frequencies, eps=1e-6, interleaved=False, scale=1.0):
    """(dx, dweight, magnitude of dweight's terms) from the formula, float64."""
    g = rope(dy, positions, frequencies, interleaved, scale, inverse=True)
    x, weight = x.double(), weight.double()
    rstd = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    unit = x * rstd
    gw = g * weight
    dx = rstd * (gw - unit * (gw * unit).mean(-1, keepdim=True))
    terms = (g * unit).flatten(0, -2)
    return dx, terms.sum(0), terms.abs().sum(0)


def activation(z, name):
    """(act(z), act'(z)) in float64."""
    z = z.double()
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp_min(0.0), (z > 0).double()
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * c * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    raise AssertionError(name)


def linear(x, weight, bias=None, act=None, residual=None):
    """(y, z) in float64."""
    z = x.double() @ weight.double().t()
    if bias is not None:
        z = z + bias.double()
    y = activation(z, act)[0]
    return (y if residual is None else y + residual.double()), z


def linear_backward(dy, x, weight, bias=None, act=None):
    """(dx, dw, dbias, dz) in float64, for 2D tensors."""
    z = linear(x, weight, bias)[1]
    dz = dy.double() * activation(z, act)[1]
    return dz @ weight.double(), dz.t() @ x.double(), dz.sum(0), dz


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """{token: logprob} of one row, float64 on the host; the four parameters already rounded to float32. One token,
    unless the draw lies on a boundary to within the rounding of a 64-bit sum: V additions in any order are good to
    V 2^-53 of the sum, here and in what is compared, so a draw within V 2^-52 of a boundary may go to either side."""
    l = logits.detach().double().cpu()
    l = torch.where(torch.isnan(l), -math.inf, l)
    top = float(l.max())
    if top == -math.inf:
        return {-1: -math.inf}
    first = int(torch.nonzero(l == top)[0, 0])
    if not temperature > 0:
        return {first: 0.0}
    if top == math.inf:
        w = (l == math.inf).double()
    else:
        w = torch.where(l == -math.inf, 0.0, torch.exp((l - top) / temperature))
    ranked = torch.argsort(l, descending=True, stable=True)
    if 0 < top_k < len(l):
        ranked = ranked[:int(top_k)]
    ws = w[ranked]
    ahead = torch.cumsum(ws, 0) - ws
    keep = ws > 0
    if top_p < 1:
        keep &= ahead <= top_p * ws.sum()
        keep[0] = True
    keep &= ws >= min(max(min_p, 0.0), 1.0)
    index = torch.sort(ranked[keep]).values
    line = torch.cumsum(w[index], 0)
    u = min(max(float(u), 0.0), 1.0) if u == u else 0.0
    room = len(l) * 2.0 ** -52 * float(line[-1])
    low, high = (min(int(torch.searchsorted(line, u * line[-1] + d, right=True)), len(index) - 1) for d in (-room, room))
    return {int(index[at]): math.log(float(w[index[at]] / line[-1])) for at in range(low, high + 1)}
