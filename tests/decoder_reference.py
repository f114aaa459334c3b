"""The operators around a decoder step's linears from their definitions, in 64 bits on the CPU, with bounds for fp32 arithmetic."""
import math

import torch

U = 2.0 ** -24   # half a unit in the last place of fp32


def _norm(v, centered, eps):
    if centered:
        v = v - v.mean(-1, keepdim=True)
    r = 1 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    return v * r, r


def _d(t):
    return None if t is None else t.detach().cpu().double()


def residual_norm(x, residual=None, weight=None, bias=None, post_weight=None, gate=None, scale=1.0, eps=1e-6, weight_offset=0.0, centered=False):
    """``(normed, stream, slack of normed, slack of stream)``.

    Sums are at most 32 additions in a thread and 10 over threads, means and roots a few roundings more: 64 u relative to the
    largest number that goes in."""
    c = 64 * U
    x, residual, weight, bias, post_weight, gate = (_d(t) for t in (x, residual, weight, bias, post_weight, gate))
    most = lambda v: v.abs().amax(-1, keepdim=True)  # noqa: E731
    b, off = x, torch.zeros(1, dtype=torch.float64)
    if post_weight is not None:
        b, r = _norm(x, centered, eps)
        w = post_weight + weight_offset
        # (the mean is off by c times the largest number; what is left of it is multiplied by r and w)
        off = (c * most(x) * r + c * b.abs()) * w.abs()
        b = b * w
    g = scale * (1.0 if gate is None else gate)
    b, off = b * g, off * (g.abs() if torch.is_tensor(g) else abs(g)) + 3 * U * (b * g).abs()
    s = b if residual is None else residual + b
    off = off + U * s.abs()
    y, r = _norm(s, centered, eps)
    # an error of the numbers goes through the norm at most twice (by itself and by the root)
    slack = 2 * most(off) * r + c * most(s) * r * centered + c * y.abs()
    w = torch.ones(1, dtype=torch.float64) if weight is None else weight + weight_offset
    y, slack = y * w, slack * w.abs() + 4 * U * (y * w).abs()
    if bias is not None:
        y, slack = y + bias, slack + U * bias.abs() + U * (y + bias).abs()
    return y, s, slack, off


ACTIVATIONS = {
    None: lambda v: v,
    "relu": lambda v: v.clamp(min=0),
    "silu": lambda v: v * torch.sigmoid(v),
    "gelu": lambda v: v * torch.special.ndtr(v),
    "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)),
}


def product(x, w, bias):
    """``(x W^T + bias, slack)``: a rounding (or a cut) for every 16 products and every slice that is added, relative to the sum
    of their magnitudes; bf16 numbers below 2^-14 lose at most 2^-25 on their way to fp16."""
    bf16 = x.dtype == torch.bfloat16
    x, w, bias = _d(x), _d(w), _d(bias)
    y, mass = x @ w.T, x.abs() @ w.abs().T
    slack = mass * (w.shape[1] / 16 + 32) * 2 * U + (w.abs().sum(1) * 2.0 ** -25 if bf16 else 0)
    if bias is not None:
        y, slack = y + bias, slack + U * (y + bias).abs()
    return y, slack


def fused(x, weights, biases, activation, residual=None, scale=1.0):
    """``(y, slack)`` of one weight, or of gate and up."""
    v, off = product(x, weights[0], biases[0])
    y = ACTIVATIONS[activation](v)
    # slopes up to 1.13; fast exponentials are off by a few u and by u for every unit of their argument (4 |v| at most)
    off = 1.13 * off + y.abs() * (16 + 8 * v.abs().clamp(max=100)) * U + 2.0 ** -126
    if len(weights) == 2:
        u, more = product(x, weights[1], biases[1])
        y, off = y * u, off * u.abs() + y.abs() * more + off * more
    y, off = y * scale, (off + 2 * U * y.abs()) * abs(scale)
    if residual is not None:
        y, off = y + _d(residual), off + U * (y + _d(residual)).abs()
    return y, off


def token_logprobs(logits, tokens, top=0, temperature=1.0):
    """``(logprobs, entropy, top tokens, top logprobs)`` of 2-D logits."""
    l, tokens = logits.detach().cpu(), tokens.detach().cpu().long()
    z = l.double() / temperature
    wrong = (z.isnan() | (z == math.inf)).any(-1)
    empty = (z == -math.inf).all(-1)
    safe = torch.where((wrong | empty)[:, None], torch.zeros_like(z), z)
    safe = safe - safe.amax(-1, keepdim=True)   # (log 6 added to a lowest bf16 number would vanish, in 64 bits too)
    every = safe.logsumexp(-1, keepdim=True)
    logp = safe - every
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    logp[empty], entropy[empty] = -math.inf, 0.0
    logp[wrong], entropy[wrong] = math.nan, math.nan
    given = logp.gather(1, tokens.clamp(0, l.shape[1] - 1)[:, None])[:, 0]
    given[tokens < 0] = 0.0
    given[tokens >= l.shape[1]] = math.nan
    order = l.double().sort(dim=-1, descending=True, stable=True).indices[:, :top]   # (NaN above all, equal ones by their index)
    return given, entropy, order, logp.gather(1, order)


def logprob_slack(vocab, logp, temperature):
    """A thread adds up at most vocab / 128 + 32 numbers, then come 12 joins; an exponential is off by 4 u and u for every unit of
    its argument, which weighs at most e^-1 of itself; the difference to the maximum and the logarithm by a few u each."""
    return (vocab / 128 + 64) * U + 8 * U * logp.abs().nan_to_num(0, 0, 0) + 16 * U
