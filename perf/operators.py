"""The attention path of a decoder layer between its quantized linears, as cases that can be timed one pass at a time.

Three operators: the norms of queries and keys with the position rotation (``norm_rotate``), the same with keys and values
written to a paged cache in 4 bits (``norm_rotate_store``, read back by ``QuantizedKVCache.load``), and attention over that
cache (``cache_attention``) with causal masks, a sliding window and first tokens that stay visible (sinks).

A case is a dict of plain values.  ``prepare`` makes what a program holds before the call, on the GPU and from the seed
alone; ``run`` is one pass, in elementary operations or (``own``) through the package's entry points; ``exact`` is the
definition in 64 bits; ``work`` is what a pass cannot do without.

The cache.  A token's keys (or values) of one head are cut into groups of 64 channels.  With lo = min(x, 0), hi = max(x, 0)
over a group: scale s = (hi - lo) / 15 rounded up to 7 significant bits, within [2^-18, 4352]; zero point z = rint(-lo / s);
code c = clamp(rint(x / s) + z, 0, 15).  The stored value is s * (c - z), exact in fp16.  NaN is stored as 0, and values
saturate at 65280.  Memory is made of slabs of 16 tokens of one head, 18 * D bytes each:

  8 D bytes   codes of the keys    [plane][token 16][t 4][j][b 2][a 4]        channel 128 plane + 32 j + 8 t + 2 a + b
  8 D bytes   codes of the values  [plane][half 2][g 8][t 4][j][odd 2][p 4]   token 8 half + 2 t + odd, channel 128 plane + 32 j + 4 g + p
  D bytes     keys:   [token 16][group] (fp16 scale, fp16 1024 + z)
  D bytes     values: [pair 8][group] (two fp16 scales, two fp16 1024 + z)

(codes are nibbles, the lower one first; planes are 128 channels, or all 64 of a head of 64).  A page holds
``page_size / 16`` slabs for each head: data[page, head, bytes].
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
MAX_SCALE, MIN_SCALE = 4352.0, 2.0 ** -18
MAX_VALUE = 15 * MAX_SCALE
POSITIONS = 32768
EPS = 1e-6


def listed():
    return [
        # A small model's layer (32 heads of 64, fp16) rotates the queries and keys of one new token: all latency.
        dict(name="rotate_1tok", kind="rotate", tokens=1, hq=32, hkv=32, d=64, rotary=64, norm=False, neighbours=False, dtype="fp16"),
        # A prompt through a grouped-query layer of the 70B shape with norms on queries and keys.
        dict(name="rotate_prompt", kind="rotate", tokens=4001, hq=64, hkv=8, d=128, rotary=128, norm=True, neighbours=False, dtype="bf16"),
        # A serving batch of 32 generates: each new token's keys and values go to its own page.
        dict(name="store_32tok", kind="store", tokens=32, hq=32, hkv=8, d=128, rotary=128, norm=True, neighbours=False, dtype="bf16", page=64),
        # A prompt of odd length with wide heads, neighbouring pairs rotated over half of the channels.
        dict(name="store_prompt", kind="store", tokens=2011, hq=16, hkv=16, d=256, rotary=128, norm=False, neighbours=True, dtype="fp16", page=32),
        # A small model answers one user: short context, the smallest attention there is.
        dict(name="attend_1x301", kind="attend", batch=1, queries=1, longest=301, ragged=False, hq=32, hkv=32, d=64, window=0, sinks=0, dtype="fp16", page=16),
        # A 7B-shaped layer (every head its own keys) for one user in the middle of a long chat.
        dict(name="attend_1x4001", kind="attend", batch=1, queries=1, longest=4001, ragged=False, hq=32, hkv=32, d=128, window=0, sinks=0, dtype="bf16", page=64),
        # The 70B shape with a serving batch whose contexts differ: the bulk of the decode work.
        dict(name="attend_32_ragged", kind="attend", batch=32, queries=1, longest=8192, ragged=True, hq=64, hkv=8, d=128, window=0, sinks=0, dtype="bf16", page=64),
        # Two users with whole books: few rows, a very long axis.
        dict(name="attend_2x131071", kind="attend", batch=2, queries=1, longest=131071, ragged=False, hq=32, hkv=8, d=128, window=0, sinks=0, dtype="fp16", page=128),
        # Sliding-window layer with wide heads and four sinks; what slid out of the window is freed.
        dict(name="attend_window", kind="attend", batch=24, queries=1, longest=16001, ragged=True, hq=16, hkv=8, d=256, window=1024, sinks=4, dtype="bf16", page=32),
        # Five drafted tokens for each of eight users are checked in one pass.
        dict(name="attend_draft", kind="attend", batch=8, queries=5, longest=4000, ragged=True, hq=32, hkv=8, d=128, window=0, sinks=0, dtype="bf16", page=64),
        # A prompt attends to itself: the largest amount of arithmetic.
        dict(name="attend_prompt", kind="attend", batch=1, queries=4096, longest=4096, ragged=False, hq=32, hkv=8, d=128, window=0, sinks=0, dtype="bf16", page=64),
        # Chunks of three prompts of other lengths behind what is in the cache already, in a window with sinks.
        dict(name="attend_chunks", kind="attend", batch=3, queries=901, longest=6007, ragged=True, hq=32, hkv=8, d=64, window=2048, sinks=4, dtype="fp16", page=48),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_once(rng):
    kind = rng.choices(("rotate", "store", "decode", "draft", "prompt"), (2, 2, 4, 1, 3))[0]
    d, dtype = rng.choice((64, 128, 128, 256)), rng.choice(("fp16", "bf16"))
    hkv = rng.choice((1, 2, 4, 5, 8, 16, 32))
    hq = hkv * rng.choice((1, 2, 5, 4, 7, 8) if hkv <= 8 else (1, 2))
    if (hq + 2 * hkv) * d == 3 << 10:   # (a row width that no model here has)
        hq += hkv
    if kind in ("rotate", "store"):
        norm = rng.random() < 0.5
        most = 4096
        if kind == "store" and norm:   # (each of a normed key's codes is one rounding away from its neighbour's)
            most = max(1, min(most, 300000 // (hkv * d)))
        case = dict(kind=kind, tokens=_log_int(rng, 1, most), hq=hq, hkv=hkv, d=d, rotary=rng.choice((d, d, d // 2, 48)), norm=norm,
                    neighbours=rng.random() < 0.3, dtype=dtype)
        if kind == "store":
            case["page"] = rng.choice((16, 32, 48, 64, 128))
        return case
    window = rng.choice((0, 0, _log_int(rng, 64, 4096)))
    sinks = rng.choice((0, 4, _log_int(rng, 1, 64))) if window else 0
    case = dict(kind="attend", hq=hq, hkv=hkv, d=d, window=window, sinks=sinks, dtype=dtype, ragged=rng.random() < 0.7, page=rng.choice((16, 32, 48, 64, 128)))
    if kind == "decode":
        case.update(batch=_log_int(rng, 1, 64), queries=1, longest=_log_int(rng, 1, 131072))
    elif kind == "draft":
        case.update(batch=_log_int(rng, 1, 32), queries=rng.randrange(2, 17), longest=_log_int(rng, 64, 16384))
    else:
        queries = _log_int(rng, 17, 4096)
        case.update(batch=rng.choice((1, 1, 2, 3)), queries=queries, longest=max(queries, _log_int(rng, 64, 8192)))
    return case


def draw(rng):
    cost = lambda c: (lambda w: max(w["bytes"], w["flops"] / 50))(work(c))  # noqa: E731
    most = max(cost(c) for c in listed())
    case = _draw_once(rng)
    while cost(case) > most or (case["kind"] == "attend" and _dense_values(case) > 1.5e9):
        case = _draw_once(rng)
    return case


def _dense_values(case):
    """Numbers in the largest padded array that a plain form makes of the case."""
    keys = case["batch"] * case["longest"] * case["hkv"] * case["d"]
    return max(keys, case["batch"] * case["hq"] * case["queries"] * case["longest"])


def _lengths(case):
    """Tokens of each sequence in the cache (its queries' own among them), and its queries."""
    if not case["ragged"]:
        return [case["longest"]] * case["batch"], [case["queries"]] * case["batch"]
    spread = [1.0] + [(0.6180339887 * i) % 1.0 for i in range(1, case["batch"])]
    lengths = [max(1, round(case["longest"] * f)) for f in spread]
    if case["queries"] == 1:
        return lengths, [1] * case["batch"]
    queries = [max(1, round(case["queries"] * (1.0 if i == 0 else 0.3 + 0.7 * f))) for i, f in enumerate(spread)]
    return [max(a, b) for a, b in zip(lengths, queries)], queries


def _dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


# ---- the cache's numbers and bytes -------------------------------------------------------------------------------

def _quantise(x):
    """Codes, scales and zero points of fp32 ``x`` [..., D], each [..., D / 64, 64 or 1]."""
    x = torch.nan_to_num(x, nan=0.0, posinf=MAX_VALUE, neginf=-MAX_VALUE).clamp(-MAX_VALUE, MAX_VALUE)
    x = x.unflatten(-1, (-1, 64))
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    s = (hi - lo) / hi.new_full((1,), 15.0)   # (a divisor on the host would become a product with its reciprocal)
    s = ((s.view(torch.int32) + 0x1FFFF) & ~0x1FFFF).view(torch.float32).clamp(MIN_SCALE, MAX_SCALE)
    z = torch.round(-lo / s).clamp(0, 15)
    return (torch.round(x / s) + z).clamp(0, 15), s, z


def _values(x):
    """What ``x`` [..., D] is once it has been stored."""
    c, s, z = _quantise(x)
    return (s * (c - z)).flatten(-2)


def _nibbles(n):
    """Bytes of codes [..., even number]."""
    n = n.to(torch.uint8).unflatten(-1, (-1, 2))
    return n[..., 0] | (n[..., 1] << 4)


def _pack(k, v):
    """The cache's bytes for fp32 keys and values [pages, heads, page, D]."""
    pages, heads, page, d = k.shape
    planes, j = max(1, d // 128), min(4, d // 32)
    c, s, z = _quantise(k)
    codes = c.reshape(pages, heads, page // 16, 16, planes, j, 4, 4, 2).permute(0, 1, 2, 4, 3, 6, 5, 8, 7)
    kc = _nibbles(codes.reshape(pages, heads, page // 16, -1))
    kp = torch.cat([s, z + 1024], -1).half().reshape(pages, heads, page // 16, -1).view(torch.uint8)
    c, s, z = _quantise(v)
    codes = c.reshape(pages, heads, page // 16, 2, 4, 2, planes, j, 8, 4).permute(0, 1, 2, 6, 3, 8, 4, 7, 5, 9)
    vc = _nibbles(codes.reshape(pages, heads, page // 16, -1))
    vp = torch.stack([s, z + 1024], -1).half().reshape(pages, heads, page // 16, 8, 2, d // 64, 2).permute(0, 1, 2, 3, 5, 6, 4)
    vp = vp.reshape(pages, heads, page // 16, -1).view(torch.uint8)
    return torch.cat([kc, vc, kp, vp], -1).reshape(pages, heads, -1)


def _unpack(data, d, page):
    """The keys and values [pages, heads, page, D] in fp32 that the cache's bytes stand for."""
    pages, heads = data.shape[:2]
    planes, j, groups = max(1, d // 128), min(4, d // 32), d // 64
    slab = data.view(pages, heads, page // 16, 18 * d)
    open_up = lambda b: torch.stack([b & 15, b >> 4], -1)  # noqa: E731
    kc = open_up(slab[..., :8 * d]).reshape(pages, heads, page // 16, planes, 16, 4, j, 2, 4).permute(0, 1, 2, 4, 3, 6, 5, 8, 7)
    kc = kc.reshape(pages, heads, page, groups, 64).float()
    kp = slab[..., 16 * d:17 * d].contiguous().view(torch.float16).reshape(pages, heads, page, groups, 2).float()
    k = (kp[..., :1] * (kc - (kp[..., 1:] - 1024))).flatten(-2)
    vc = open_up(slab[..., 8 * d:16 * d]).reshape(pages, heads, page // 16, planes, 2, 8, 4, j, 2, 4).permute(0, 1, 2, 4, 6, 8, 3, 7, 5, 9)
    vc = vc.reshape(pages, heads, page, groups, 64).float()
    vp = slab[..., 17 * d:].contiguous().view(torch.float16).reshape(pages, heads, page // 16, 8, groups, 2, 2).permute(0, 1, 2, 3, 6, 4, 5)
    vp = vp.reshape(pages, heads, page, groups, 2).float()
    v = (vp[..., :1] * (vc - (vp[..., 1:] - 1024))).flatten(-2)
    return k, v


# ---- inputs ------------------------------------------------------------------------------------------------------

def _table(rotary):
    """cos | sin of every position's angles, fp32 [POSITIONS, rotary]."""
    freq = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEVICE) / rotary)
    angle = torch.arange(POSITIONS, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], -1).float()


def _prepare_tokens(case, gen):
    t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
    # the row of a fused q/k/v linear: queries, keys and values are views of it
    x = torch.randn(t, (hq + 2 * hkv) * d, generator=gen, device=DEVICE).to(_dtype(case))
    q, k, v = x.split([hq * d, hkv * d, hkv * d], -1)
    weight = lambda: (1 + 0.1 * torch.randn(d, generator=gen, device=DEVICE)).to(_dtype(case)) if case["norm"] else None  # noqa: E731
    state = dict(case=case, q=q.unflatten(-1, (hq, d)), k=k.unflatten(-1, (hkv, d)), v=v.unflatten(-1, (hkv, d)), table=_table(case["rotary"]),
                 positions=torch.randint(0, POSITIONS, (t,), generator=gen, device=DEVICE), q_weight=weight(), k_weight=weight())
    if case["kind"] == "store":
        page = case["page"]
        if t < 256:   # decode: every token in a sequence, and so in a page, of its own
            pages = t
            state["slots"] = torch.randperm(pages, generator=gen, device=DEVICE) * page + torch.randint(0, page, (t,), generator=gen, device=DEVICE)
        else:         # a prompt: whole pages in any order, the first one begun by someone else's prefix
            pages = -(-t // page) + 1
            at = torch.arange(t, device=DEVICE) + 5
            state["slots"] = torch.randperm(pages, generator=gen, device=DEVICE)[at // page] * page + at % page
        state["data"] = torch.zeros(pages, hkv, page // 16 * 18 * d, dtype=torch.uint8, device=DEVICE)
    return state


def _prepare_attend(case, gen):
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    lengths, queries = _lengths(case)
    need = [-(-n // page) for n in lengths]
    pages = sum(need)
    k = torch.randn(pages, hkv, page, d, generator=gen, device=DEVICE)
    v = torch.randn(pages, hkv, page, d, generator=gen, device=DEVICE)
    # queries share a direction, and the first token's key lies along it: the weight that first tokens draw
    lean = 0.4 * torch.randn(hkv, d, generator=gen, device=DEVICE)
    q = torch.randn(sum(queries), hkv, hq // hkv, d, generator=gen, device=DEVICE) + lean[:, None]
    order = torch.randperm(pages, generator=gen, device=DEVICE).int()
    table = torch.full((case["batch"], max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        k[order[at].long(), :, 0] = 2 * lean
        if case["window"]:   # pages that no query sees any more are not the sequence's
            first = max(0, lengths[b] - queries[b] - case["window"] + 1) // page
            kept = -(-case["sinks"] // page)
            if first > kept:
                table[b, kept:first] = -1
        at += n
    state = dict(case=case, data=_pack(k, v), q=q.reshape(-1, hq, d).to(_dtype(case)), table=table,
                 lengths=torch.tensor(lengths, dtype=torch.int32, device=DEVICE), queries=None)
    if case["ragged"] and case["queries"] > 1:
        starts = [0]
        for n in queries:
            starts.append(starts[-1] + n)
        state["queries"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return _prepare_attend(case, gen) if case["kind"] == "attend" else _prepare_tokens(case, gen)


# ---- one pass ----------------------------------------------------------------------------------------------------

def _rotated(x, weight, state):
    """fp32 norm and rotation of ``x`` [tokens, heads, D]."""
    rotary = state["case"]["rotary"]
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    cs = state["table"][state["positions"]][:, None]
    cos, sin = cs[..., :rotary // 2], cs[..., rotary // 2:]
    if state["case"]["neighbours"]:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _run_tokens(state):
    case, dtype = state["case"], state["q"].dtype
    q = _rotated(state["q"], state["q_weight"], state)
    k = _rotated(state["k"], state["k_weight"], state)
    if case["kind"] == "rotate":
        return q.to(dtype), k.to(dtype)
    return q.to(dtype), _values(k).to(dtype), _values(state["v"].float()).to(dtype)


def _run_attend(state):
    case, q = state["case"], state["q"]
    hq, hkv, d, page, batch = case["hq"], case["hkv"], case["d"], case["page"], case["batch"]
    lengths = state["lengths"].long()
    if state["queries"] is None:
        count = torch.full_like(lengths, q.shape[0] // batch)
        first = torch.arange(batch, device=q.device) * (q.shape[0] // batch)
    else:
        starts = state["queries"].long()
        first, count = starts[:-1], starts[1:] - starts[:-1]
    most = case["queries"]
    # sequences side by side, padded to the longest: queries [batch, hkv, most * r, D], keys and values [batch, hkv, keys, D]
    turn = torch.arange(most, device=q.device)
    row = (first[:, None] + turn).clamp(max=q.shape[0] - 1)
    qs = q[row].float().unflatten(2, (hkv, hq // hkv)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    table = state["table"].long().clamp(min=0)
    k, v = (x[table].permute(0, 2, 1, 3, 4).flatten(2, 3) for x in _unpack(state["data"], d, page))
    key = torch.arange(k.shape[2], device=q.device)
    position = (lengths - count)[:, None] + turn
    seen = key <= position[..., None]
    if case["window"]:
        seen = seen & ((key > position[..., None] - case["window"]) | (key < case["sinks"]))
    seen = (seen & (turn < count[:, None])[..., None]).repeat_interleave(hq // hkv, 1)[:, None]
    scores = (qs @ k.transpose(-1, -2)) * (d ** -0.5)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    out = (weight @ v) / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = out.unflatten(2, (most, hq // hkv)).permute(0, 2, 1, 3, 4).reshape(batch * most, hq, d).to(q.dtype)
    if state["queries"] is None:
        return out
    return out[torch.nonzero((turn < count[:, None]).flatten())[:, 0]]


def _run_own(state):
    import atlasinfer_b200 as ab

    case = state["case"]
    if case["kind"] != "rotate" and "cache" not in state:   # the handle that a program keeps
        state["cache"] = ab.QuantizedKVCache(state["data"].shape[0], case["hkv"], case["d"], page_size=case["page"], data=state["data"])
    if case["kind"] == "attend":
        return ab.cache_attention(state["q"], state["cache"], state["table"], state["lengths"], query_starts=state["queries"],
                                  max_queries=case["queries"], window=case["window"] or None, sinks=case["sinks"])
    how = dict(q_weight=state["q_weight"], k_weight=state["k_weight"], eps=EPS, interleaved=case["neighbours"])
    if case["kind"] == "rotate":
        return ab.norm_rotate(state["q"], state["k"], state["table"], state["positions"], **how)
    q = ab.norm_rotate_store(state["q"], state["k"], state["v"], state["cache"], state["slots"], state["table"], state["positions"], **how)
    k, v = state["cache"].load(state["slots"], dtype=q.dtype)
    return q, k, v


def run(state):
    if own:
        return _run_own(state)
    return _run_attend(state) if state["case"]["kind"] == "attend" else _run_tokens(state)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def _exact_turned(x, weight, state):
    x = x.double()
    d, rotary = x.shape[-1], state["case"]["rotary"]
    if weight is not None:
        x = x / ((x * x).sum(-1, keepdim=True) / d + EPS).sqrt() * weight.double()
    i = torch.arange(rotary // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if state["case"]["neighbours"] else (i, i + rotary // 2)
    angles = state["table"].double().index_select(0, state["positions"])
    point = torch.complex(x[..., a], x[..., b]) * torch.complex(angles[:, None, i], angles[:, None, i + rotary // 2])
    y = x.clone()
    y[..., a], y[..., b] = point.real, point.imag
    return y


def _exact_stored(x):
    x = x.double()
    x = torch.where(x.isnan(), torch.zeros_like(x), x).clamp(-MAX_VALUE, MAX_VALUE)
    parts = x.split(64, -1)
    stored = []
    for part in parts:
        low, high = part.min(-1, keepdim=True).values.clamp(max=0), part.max(-1, keepdim=True).values.clamp(min=0)
        mantissa, exponent = torch.frexp((high - low) / 15)
        s = torch.ldexp(torch.ceil(mantissa * 128) / 128, exponent).clamp(MIN_SCALE, MAX_SCALE)
        z = (-low / s).round()
        stored.append(((part / s).round() + z).clamp(0, 15).sub(z) * s)
    return torch.cat(stored, -1)


def _exact_cache(data, pages, head, d, page):
    """Keys and values [tokens, D] in 64 bits of one head in a list of pages, each number by its place among the bytes."""
    dev = data.device
    token = torch.arange(page, device=dev)
    slab, tok = (token // 16 * 18 * d)[:, None], (token % 16)[:, None]
    ch = torch.arange(d, device=dev)[None]
    plane, wide = ch // 128, min(d, 128)
    words = wide // 32
    block = data[pages, head].to(torch.int64)
    half = lambda at: (block[:, at] | (block[:, at + 1] << 8)).to(torch.int16).view(torch.float16).double()  # noqa: E731
    c = ch % wide
    nib = (((tok * 4 + c % 32 // 8) * words + c // 32) * 2 + c % 2) * 4 + c % 8 // 2 + plane * 16 * wide
    at = slab + nib // 2
    code = (block[:, at] >> (4 * (nib % 2))) & 15
    p = slab + 16 * d + (tok * (d // 64) + ch // 64) * 4
    k = half(p) * (code - (half(p + 2) - 1024))
    unit = (((tok // 8 * 8 + c % 32 // 4) * 4 + tok % 8 // 2) * words + c // 32) * 2 + tok % 2
    nib = unit * 4 + c % 4 + plane * 16 * wide
    at = slab + 8 * d + nib // 2
    code = (block[:, at] >> (4 * (nib % 2))) & 15
    p = slab + 17 * d + (tok // 2 * (d // 64) + ch // 64) * 8 + tok % 2 * 2
    v = half(p) * (code - (half(p + 4) - 1024))
    return k.flatten(0, 1), v.flatten(0, 1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] != "attend":
        q, k = _exact_turned(state["q"], state["q_weight"], state), _exact_turned(state["k"], state["k_weight"], state)
        return (q, k) if case["kind"] == "rotate" else (q, _exact_stored(k), _exact_stored(state["v"]))
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    lengths, queries = _lengths(case)
    out = torch.zeros(sum(queries), hq, d, dtype=torch.float64, device=DEVICE)
    begin = 0
    for b, (length, count) in enumerate(zip(lengths, queries)):
        pages = state["table"][b, :-(-length // page)].long().clamp(min=0)
        key = torch.arange(length, device=DEVICE)
        position = length - count + torch.arange(count, device=DEVICE)[:, None]
        hidden = key > position
        if case["window"]:
            hidden |= (key <= position - case["window"]) & (key >= case["sinks"])
        for h in range(hkv):
            k, v = _exact_cache(state["data"], pages, h, d, page)
            for n in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                s = state["q"][begin:begin + count, n].double() @ k[:length].T / math.sqrt(d)
                out[begin:begin + count, n] = torch.softmax(s.masked_fill_(hidden, -math.inf), -1) @ v[:length]
        begin += count
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    """Bytes: inputs, outputs and what is visible of the cache, once.  Operations: products and sums of the formulas."""
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] != "attend":
        t = case["tokens"]
        nbytes = t * (2 * (hq + hkv) * d + 4 * case["rotary"] + 8 + 2 * hq * d)
        if case["kind"] == "rotate":
            nbytes += t * 2 * hkv * d
        else:   # v read, the cache written, and what was stored read back and returned
            nbytes += t * (2 * hkv * d + 8 + 2 * 18 * d // 16 * hkv + 4 * hkv * d)
        return dict(bytes=float(nbytes), flops=float(t * (hq + hkv) * d * 8))
    nbytes = flops = 0.0
    for length, count in zip(*_lengths(case)):
        first, last = length - count, length - 1
        if case["window"]:
            w, s = case["window"], case["sinks"]
            start = max(0, first - w + 1)
            tokens = length - start + min(s, start)
            pairs = sum(min(p + 1, w + min(s, max(0, p + 1 - w))) for p in range(first, last + 1))
        else:
            tokens, pairs = length, (first + 1 + last + 1) * count // 2
        nbytes += tokens * hkv * 18 * d / 16 + 4.0 * count * hq * d
        flops += 4.0 * d * hq * pairs
    return dict(bytes=nbytes, flops=flops)
