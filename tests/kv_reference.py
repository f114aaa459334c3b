"""Queries, keys and the 4-bit cache from their definitions, in 64 bits on the CPU."""
import math

import torch

MAX_SCALE, MIN_SCALE = 4352.0, 2.0 ** -18
# half a unit in the last place, relative
HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def groups(x):
    """(codes, scale, zero point) of ``x`` [..., D]: [..., D / 64, 64], [..., D / 64, 1] twice."""
    x = x.detach().cpu().double()
    x = torch.where(x.isnan(), torch.zeros_like(x), x).clamp(-15 * MAX_SCALE, 15 * MAX_SCALE).unflatten(-1, (-1, 64))
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    m, e = torch.frexp((hi - lo) / 15)
    s = torch.ldexp(torch.ceil(m * 128) / 128, e).clamp(MIN_SCALE, MAX_SCALE)
    z = (-lo / s).round().clamp(0, 15)
    return ((x / s).round() + z).clamp(0, 15), s, z


def stored(x):
    c, s, z = groups(x)
    return (s * (c - z)).flatten(-2)


def steps(x):
    """The step of every number of ``x``."""
    _, s, _ = groups(x)
    return s.expand(*s.shape[:-1], 64).flatten(-2)


def turned(x, weight=None, table=None, positions=None, eps=1e-6, weight_offset=0.0, interleaved=False):
    x = x.detach().cpu().double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (weight.cpu().double() + weight_offset)
    if table is None:
        return x
    rotary = table.shape[1]
    cs = table.cpu().double()[positions.cpu().long()][:, None]
    cos, sin = cs[..., :rotary // 2], cs[..., rotary // 2:]
    y = x.clone()
    a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def attention(q, ks, vs, queries, window=None, sinks=0, scale=None):
    """``(out, mass)`` for stored keys and values of every sequence (lists of [tokens, kv_heads, D], in 64 bits); ``mass`` is
    the weighted mean of |v|, what an error of the weights is relative to."""
    q = q.detach().cpu().double()
    total, heads, d = q.shape
    out, mass = torch.zeros_like(q), torch.zeros_like(q)
    begin = 0
    for k, v, n in zip(ks, vs, queries):
        length, kv_heads = k.shape[:2]
        r = heads // kv_heads
        x = q[begin:begin + n].unflatten(1, (kv_heads, r))
        key, position = torch.arange(length), length - n + torch.arange(n)[:, None]
        seen = key <= position
        if window is not None:
            seen &= (key > position - window) | (key < sinks)
        s = torch.einsum("nhrd,khd->nhrk", x, k) * (d ** -0.5 if scale is None else scale)
        s = s.masked_fill(~seen[:, None, None], -math.inf)
        top = s.amax(-1, keepdim=True) if length else torch.zeros(n, kv_heads, r, 1, dtype=torch.float64)
        p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        out[begin:begin + n] = torch.einsum("nhrk,khd->nhrd", p, v).flatten(1, 2)
        mass[begin:begin + n] = torch.einsum("nhrk,khd->nhrd", p, v.abs()).flatten(1, 2)
        begin += n
    return out, mass


def assert_rounded(got, want, slack, what=""):
    """``got`` is ``want`` rounded to its type, but for an error of ``slack`` (a tensor or a number) before the rounding."""
    u = HALF_ULP[got.dtype]
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -134   # half the spacing of the smallest numbers
    got = got.detach().cpu().double()
    err, most = (got - want).abs(), want.abs() * u + tiny + slack * (1 + u)
    bad = ~(err <= most)
    assert not bad.any(), f"{what}{int(bad.sum())} of {bad.numel()} off, worst {float((err / most).nan_to_num(9e9).max()):.3g} times the bound"
