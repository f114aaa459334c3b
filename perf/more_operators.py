"""What a decoder step computes around its quantized linears, as cases that can be timed one pass at a time.

Three kinds of operators, from the stream of hidden rows to the answer:

* ``norm``    ``residual_norm``: a block's output is normed (or not), gated, scaled and added to the stream, and the sum is
  normed for the next block, by its root mean square or (``centered``) by mean and variance
* ``linear``  ``linear_epilogue`` and ``gated_linear``: products with quantized weights whose bias, activation, product with a
  second linear, scale and residual are part of the pass
* ``answer``  ``token_logprobs``: log probabilities of given tokens, the entropy of every row, and its likeliest tokens

A case is a dict of plain values.  ``prepare`` makes what a program holds before the call, on the GPU and from the seed
alone; ``run`` is one pass, in elementary operations or (``own``) through the package's entry points; ``exact`` is the
definition in 64 bits; ``work`` is what a pass cannot do without.

A quantized weight [N, K] has an int8 code for every number, an fp16 scale for every ``block`` numbers of a row, and outliers
that stand for themselves: W = fp16(code * scale), or the outlier.  Its streams hold the codes of the others back to back, the
outliers and their flat positions, and the scales.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
ACTIVATIONS = ("relu", "silu", "gelu", "gelu_tanh")


def listed():
    return [
        # One user, one token: the norm in front of a block of the 7B shape, all latency.
        dict(name="norm_1tok", kind="norm", tokens=1, hidden=4096, centered=False, post=False, gate="none", stream="same", dtype="bf16"),
        # A batch of odd length and width: norms on both sides of a block, gates of each row, a stream in 32 bits, means taken out.
        dict(name="norm_ragged", kind="norm", tokens=515, hidden=5001, centered=True, post=True, gate="rows", stream="fp32", dtype="fp16"),
        # A prompt of the 70B shape: the traffic of the whole stream.
        dict(name="norm_prompt", kind="norm", tokens=4096, hidden=8192, centered=False, post=False, gate="none", stream="same", dtype="bf16"),
        # One token through the 7B shape's down projection, added to the stream.
        dict(name="residual_1tok", kind="linear", tokens=1, n=4096, k=11008, block=128, gated=False, act="none", bias=False, residual=True, dtype="bf16"),
        # The first linear of an OPT-1.3B block for a batch of 24, with bias and relu.
        dict(name="relu_24tok", kind="linear", tokens=24, n=8192, k=2048, block=128, gated=False, act="relu", bias=True, residual=False, dtype="fp16"),
        # One token through gate and up of the 7B shape.
        dict(name="gated_1tok", kind="linear", tokens=1, n=11008, k=4096, block=128, gated=True, act="silu", bias=False, residual=False, dtype="bf16"),
        # A serving batch through gate and up of the 70B shape: the most weights there are.
        dict(name="gated_32tok", kind="linear", tokens=32, n=28672, k=8192, block=128, gated=True, act="silu", bias=False, residual=False, dtype="bf16"),
        # A prompt of odd length through a down projection, scaled and added to the stream.
        dict(name="residual_prompt", kind="linear", tokens=1001, n=4096, k=11008, block=64, gated=False, act="none", bias=True, residual=True, dtype="fp16"),
        # A long prompt through gate and up of the 7B shape: the most arithmetic.
        dict(name="gated_prompt", kind="linear", tokens=2048, n=11008, k=4096, block=128, gated=True, act="gelu_tanh", bias=False, residual=False, dtype="bf16"),
        # One user's next token from OPT's vocabulary, with its five likeliest.
        dict(name="answer_1", kind="answer", rows=1, vocab=50272, top=5, temperature=1.0, masked=0.0, dtype="fp16"),
        # A serving batch over a large vocabulary of odd size, part of it masked, with twenty alternatives each.
        dict(name="answer_64", kind="answer", rows=64, vocab=128257, top=20, temperature=0.7, masked=0.3, dtype="bf16"),
        # A long text is scored: only its own tokens' probabilities and the entropies.
        dict(name="score_2048", kind="answer", rows=2048, vocab=50272, top=0, temperature=1.0, masked=0.0, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_once(rng):
    kind = rng.choices(("norm", "linear", "answer"), (3, 4, 3))[0]
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "norm":
        hidden = _log_int(rng, 33, 16384)
        return dict(kind=kind, tokens=_log_int(rng, 1, 8192), hidden=hidden if rng.random() < 0.3 else -(-hidden // 64) * 64, centered=rng.random() < 0.4,
                    post=rng.random() < 0.4, gate=rng.choice(("none", "none", "channels", "rows")), stream=rng.choice(("same", "same", "fp32", "none")), dtype=dtype)
    if kind == "linear":
        gated, block = rng.random() < 0.5, rng.choice((32, 64, 128, 128))
        n, k = _log_int(rng, 64, 28672), _log_int(rng, 256, 16384)
        return dict(kind=kind, tokens=_log_int(rng, 1, 2048), n=n if rng.random() < 0.3 else -(-n // 16) * 16, k=-(-k // 128) * 128, block=block, gated=gated,
                    act=rng.choice(ACTIVATIONS) if gated else rng.choice(("none",) + ACTIVATIONS), bias=rng.random() < 0.4, residual=rng.random() < 0.5, dtype=dtype)
    return dict(kind=kind, rows=_log_int(rng, 1, 2048), vocab=_log_int(rng, 500, 262144), top=rng.choice((0, 1, 5, 20, rng.randrange(1, 33))),
                temperature=rng.choice((1.0, 1.0, 0.7, 1.5)), masked=rng.choice((0.0, 0.0, 0.3, 0.97)), dtype=rng.choice((dtype, dtype, "fp32")))


def draw(rng):
    cost = lambda c: (lambda w: max(w["bytes"], w["flops"] / 50))(work(c))  # noqa: E731
    most = max(cost(c) for c in listed())
    case = _draw_once(rng)
    while cost(case) > most:
        case = _draw_once(rng)
    return case


def _dtype(name):
    return {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}[name]


# ---- inputs ------------------------------------------------------------------------------------------------------

def _prepare_norm(case, gen):
    t, h, dtype = case["tokens"], case["hidden"], _dtype(case["dtype"])
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=DEVICE)  # noqa: E731
    stream = None
    if case["stream"] != "none":
        # a few channels of a stream are far larger than the others, in every token
        loud = 1 + 30 * (torch.rand(h, generator=gen, device=DEVICE) < 0.004)
        stream = (2 * randn(t, h) * loud).to(torch.float32 if case["stream"] == "fp32" else dtype)
    gate = {"none": lambda: None, "channels": lambda: (0.5 + 0.2 * randn(h)).to(dtype), "rows": lambda: (0.5 + 0.2 * randn(t, h)).to(dtype)}[case["gate"]]()
    return dict(case=case, x=(randn(t, h) + 0.1).to(dtype), residual=stream, gate=gate, scale=0.5 if case["gate"] == "channels" else 1.0,
                weight=(1 + 0.1 * randn(h)).to(dtype), bias=(0.1 * randn(h)).to(dtype) if case["centered"] else None,
                post_weight=(1 + 0.1 * randn(h)).to(dtype) if case["post"] else None)


def _weight(n, k, block, gen):
    """A random weight's codes [N, K], scales [N, K / block] and outliers (flat positions, values), by blocks: what is further
    than three deviations from a block's mean stands for itself, the others are rounded to 127ths of their largest."""
    w = torch.randn(n, k // block, block, generator=gen, device=DEVICE) * 0.02
    far = torch.arange(w.numel() // 1000, device=DEVICE) * 1000   # (one in a thousand, no place twice)
    far += torch.randint(0, 1000, far.shape, generator=gen, device=DEVICE)
    w.view(-1)[far] = torch.rand(far.shape, generator=gen, device=DEVICE) * 0.8 - 0.4
    w = w.half()
    wide = w.float()
    outlier = (wide - wide.mean(-1, keepdim=True)).abs() > 3 * wide.std(-1, keepdim=True)
    scale = wide.masked_fill(outlier, 0).abs().amax(-1, keepdim=True).div(127).half()
    codes = (wide / scale.float()).round().clamp(-127, 127).masked_fill(outlier | (scale == 0), 0).to(torch.int8)
    where = outlier.flatten().nonzero().flatten()
    return dict(codes=codes.view(n, k), scales=scale.view(n, -1), outliers=w.flatten()[where], where=where, stream=codes.flatten()[~outlier.flatten()])


def _prepare_linear(case, gen):
    t, n, k, dtype = case["tokens"], case["n"], case["k"], _dtype(case["dtype"])
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=DEVICE)  # noqa: E731
    count = 2 if case["gated"] else 1
    return dict(case=case, x=randn(t, k).to(dtype), weights=[_weight(n, k, case["block"], gen) for _ in range(count)],
                biases=[(0.1 * randn(n)).half() if case["bias"] else None for _ in range(count)], residual=randn(t, n).to(dtype) if case["residual"] else None,
                scale=0.5 if case["residual"] and case["bias"] else 1.0)


def _prepare_answer(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    sharp = 0.5 + 3 * torch.rand(rows, 1, generator=gen, device=DEVICE)
    logits = torch.randn(rows, vocab, generator=gen, device=DEVICE) * sharp
    if case["masked"]:   # tokens that a grammar rules out; it may rule all of them out
        logits.masked_fill_(torch.rand(rows, vocab, generator=gen, device=DEVICE) < case["masked"], -math.inf)
        if rows > 2:
            logits[rows // 2] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE)
    likely = logits.argmax(-1)
    tokens = torch.where(torch.rand(rows, generator=gen, device=DEVICE) < 0.6, likely, tokens)
    if rows > 4:
        tokens[-1] = -1   # a place in the batch without a token
    return dict(case=case, logits=logits.to(_dtype(case["dtype"])), tokens=tokens)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return dict(norm=_prepare_norm, linear=_prepare_linear, answer=_prepare_answer)[case["kind"]](case, gen)


# ---- one pass ----------------------------------------------------------------------------------------------------

def _normed(x, centered):
    if centered:
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _run_norm(state):
    case, x = state["case"], state["x"]
    block = x.float()
    if state["post_weight"] is not None:
        block = _normed(block, case["centered"]) * state["post_weight"].float()
    if state["gate"] is not None:
        block = block * state["gate"].float()
    block = block * state["scale"]
    residual = state["residual"]
    stream = block if residual is None else residual.float() + block
    normed = _normed(stream, case["centered"]) * state["weight"].float()
    if state["bias"] is not None:
        normed = normed + state["bias"].float()
    return dict(normed=normed.to(x.dtype), stream=stream.to(x.dtype if residual is None else residual.dtype))


def _activated(x, act):
    if act == "relu":
        return x.clamp(min=0)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * 2 ** -0.5))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x


def _product(state, i):
    """x W^T + bias in 32 bits."""
    weight, block = state["weights"][i], state["case"]["block"]
    w = (weight["codes"].half().unflatten(-1, (-1, block)) * weight["scales"][..., None]).flatten()
    w[weight["where"]] = weight["outliers"]
    y = state["x"].float() @ w.view(weight["codes"].shape).float().T
    return y if state["biases"][i] is None else y + state["biases"][i].float()


def _run_linear(state):
    case = state["case"]
    y = _activated(_product(state, 0), case["act"])
    if case["gated"]:
        y = y * _product(state, 1)
    y = y * state["scale"]
    if state["residual"] is not None:
        y = state["residual"].float() + y
    return dict(y=y.to(state["x"].dtype))


def _run_answer(state):
    case, logits, tokens = state["case"], state["logits"].float(), state["tokens"]
    top = logits.amax(-1, keepdim=True)
    nothing = top[:, 0] == -math.inf   # no token can follow
    away = (logits - torch.where(top == -math.inf, 0.0, top)) / case["temperature"]
    weight = torch.exp(away)
    total = weight.sum(-1, dtype=torch.float64)
    log_total = total.log().float()
    mean = (weight * away.masked_fill(away == -math.inf, 0.0)).sum(-1, dtype=torch.float64) / total
    given = away.gather(1, tokens.clamp(min=0)[:, None])[:, 0] - log_total
    given = torch.where(nothing, -math.inf, given)
    found = dict(logprobs=torch.where(tokens < 0, 0.0, given), entropy=torch.where(nothing, 0.0, (total.log() - mean).float()))
    if case["top"]:
        order = state["logits"].sort(dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        found.update(top_tokens=order, top_logprobs=torch.where(nothing[:, None], -math.inf, away.gather(1, order) - log_total[:, None]))
    return found


def _run_own(state):
    import atlasinfer_b200 as ab

    case = state["case"]
    if case["kind"] == "norm":
        normed, stream = ab.residual_norm(state["x"], state["residual"], state["weight"], state["bias"], post_weight=state["post_weight"], gate=state["gate"],
                                          scale=state["scale"], eps=EPS, centered=case["centered"])
        return dict(normed=normed, stream=stream)
    if case["kind"] == "answer":
        found = ab.token_logprobs(state["logits"], state["tokens"], top=case["top"], temperature=case["temperature"])
        answer = dict(logprobs=found.logprobs, entropy=found.entropy)
        if case["top"]:
            answer.update(top_tokens=found.top_tokens, top_logprobs=found.top_logprobs)
        return answer
    if "linears" not in state:   # the modules that a program keeps; as in a model, gate and up are joined
        state["linears"] = [ab.QuantizedLinear(ab.QuantizedTensor(w["stream"], w["outliers"], w["where"], w["scales"].flatten(), torch.Size(w["codes"].shape),
                                                                  case["block"]), b) for w, b in zip(state["weights"], state["biases"])]
        if case["gated"]:
            ab.fuse_linears(state["linears"])
    how = dict(activation=None if case["act"] == "none" else case["act"], residual=state["residual"], scale=state["scale"])
    if case["gated"]:
        return dict(y=ab.gated_linear(*state["linears"], state["x"], **how))
    return dict(y=ab.linear_epilogue(state["linears"][0], state["x"], **how))


def run(state):
    if own:
        return _run_own(state)
    return dict(norm=_run_norm, linear=_run_linear, answer=_run_answer)[state["case"]["kind"]](state)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def _exact_normed(x, weight, bias, centered):
    mean = x.sum(-1, keepdim=True) / x.shape[-1] if centered else 0.0
    spread = ((x - mean) ** 2).sum(-1, keepdim=True) / x.shape[-1]
    y = (x - mean) / (spread + EPS).sqrt() * weight.double()
    return y if bias is None else y + bias.double()


def _exact_norm(state, case):
    added = state["x"].double()
    if case["post"]:
        added = _exact_normed(added, state["post_weight"], None, case["centered"])
    added = added * state["scale"] * (1.0 if state["gate"] is None else state["gate"].double())
    stream = added if state["residual"] is None else added + state["residual"].double()
    return dict(normed=_exact_normed(stream, state["weight"], state["bias"], case["centered"]), stream=stream)


def _exact_linear(state, case):
    parts = []
    for weight, bias in zip(state["weights"], state["biases"]):
        wide = torch.repeat_interleave(weight["scales"].double(), case["block"], -1).mul_(weight["codes"]).half().double()
        wide.view(-1).index_copy_(0, weight["where"], weight["outliers"].double())
        parts.append(torch.addmm(torch.zeros(case["n"], dtype=torch.float64, device=DEVICE) if bias is None else bias.double(), state["x"].double(), wide.T))
        del wide
    y = parts[0]
    y = dict(none=lambda: y, relu=lambda: torch.relu(y), silu=lambda: y * torch.sigmoid(y), gelu=lambda: y * torch.special.ndtr(y),
             gelu_tanh=lambda: y * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * y * (1 + 0.044715 * y * y)))[case["act"]]()
    for other in parts[1:]:
        y = y * other
    return dict(y=y * state["scale"] + (0.0 if state["residual"] is None else state["residual"].double()))


def _exact_answer(state, case):
    z = state["logits"].double() / case["temperature"]
    every = z.logsumexp(-1, keepdim=True)
    empty = every[:, 0] == -math.inf
    logp = torch.where(empty[:, None], -math.inf, z - every)
    chance = logp.exp()
    at = torch.arange(z.shape[0], device=DEVICE)
    found = dict(logprobs=torch.where(state["tokens"] >= 0, logp[at, state["tokens"]], 0.0),
                 entropy=-torch.where(chance > 0, chance * logp, 0.0).sum(-1))
    if case["top"]:
        ranked = z.sort(dim=-1, descending=True, stable=True)[1][:, :case["top"]]
        found.update(top_tokens=ranked, top_logprobs=logp[at[:, None], ranked])
    return found


def exact(case, seed):
    return dict(norm=_exact_norm, linear=_exact_linear, answer=_exact_answer)[case["kind"]](prepare(case, seed), case)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    """Bytes: inputs and outputs once.  Operations: products and sums of the formulas."""
    if case["kind"] == "norm":
        t, h = case["tokens"], case["hidden"]
        wide = {"same": 2, "fp32": 4, "none": 0}[case["stream"]]
        nbytes = t * h * (4 + wide + (wide or 2)) + {"none": 0, "channels": 2 * h, "rows": 2 * t * h}[case["gate"]] + 2 * h * (1 + case["post"] + case["centered"])
        return dict(bytes=float(nbytes), flops=float(t * h * (8 + 5 * case["post"])))
    if case["kind"] == "linear":
        t, n, k = case["tokens"], case["n"], case["k"]
        count = 1 + case["gated"]
        weights = count * (n * k + 2 * n * k / case["block"] + 0.004 * n * k * 4 + 2 * n * case["bias"])
        return dict(bytes=float(weights + 2 * t * k + 2 * t * n * (1 + case["residual"])), flops=float(2 * t * n * k * count + 8 * t * n))
    rows, vocab = case["rows"], case["vocab"]
    return dict(bytes=float(rows * (vocab * (4 if case["dtype"] == "fp32" else 2) + 16 + 12 * case["top"])), flops=float(rows * vocab * 6))
