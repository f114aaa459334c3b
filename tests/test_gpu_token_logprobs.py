"""Log probabilities of tokens, entropies and likeliest tokens against their definition in 64 bits."""
import math

import pytest
import torch

import atlasinfer_b200 as ab

from . import decoder_reference as D

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def logits_of(rows, vocab, dtype, seed, device, scale=3.0):
    return (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


def check(logits, tokens, top=0, temperature=1.0):
    got = ab.token_logprobs(logits, tokens, top=top, temperature=temperature)
    flat = logits.reshape(-1, logits.shape[-1])
    lp, h, order, tops = D.token_logprobs(flat, tokens.reshape(-1), top, temperature)
    vocab = flat.shape[1]
    assert got.logprobs.shape == got.entropy.shape == tokens.shape and got.logprobs.dtype == F32
    assert got.top_tokens.shape == got.top_logprobs.shape == (*tokens.shape, top) and got.top_tokens.dtype == torch.int64
    assert torch.equal(got.top_tokens.cpu().reshape(order.shape), order)
    for name, a, b in (("logprobs", got.logprobs, lp), ("top", got.top_logprobs, tops)):
        a, b = a.cpu().double().reshape(b.shape), b.float().double()   # (the lowest bf16 number at temperature 0.5 is beyond fp32: -inf)
        same = (a == b) | (a.isnan() & b.isnan())
        bad = ~(same | ((a - b).abs() <= D.logprob_slack(vocab, b, temperature)))
        assert not bad.any(), (name, a[bad][:5], b[bad][:5])
    a = got.entropy.cpu().double().reshape(-1)
    # the sum of e d is off as the sum of e is, relative to itself, which is at most entropy + 1
    bad = ~((a.isnan() & h.isnan()) | ((a - h).abs() <= 3 * (1 + h) * D.logprob_slack(vocab, h, temperature)))
    assert not bad.any(), ("entropy", a[bad][:5], h[bad][:5])


@pytest.mark.parametrize("dtype", (F16, BF16, F32))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 5), (3, 31), (1, 1000), (5, 4097), (2, 50272), (1, 131073), (40, 777), (200, 64), (3, 8192), (2, 32001), (64, 33001), (1, 24), (9, 20007)])
def test_shapes(cuda_device, rows, vocab, dtype):
    logits = logits_of(rows, vocab, dtype, rows, cuda_device)
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(1)).to(torch.int32 if rows % 2 else torch.int64).to(cuda_device)
    for top in sorted({0, 1, min(5, vocab), min(32, vocab)}):
        check(logits, tokens, top, 1.0 if top else 0.6)


def test_every_top(cuda_device):
    logits, tokens = logits_of(7, 3000, BF16, 3, cuda_device), torch.arange(7, device=cuda_device)
    for top in range(33):
        check(logits, tokens, top, 1.3)


@pytest.mark.parametrize("dtype", (F16, BF16, F32))
@pytest.mark.parametrize("v", (300, 9001, 60001))
def test_ties_and_orders(cuda_device, dtype, v):
    """Rows of one number, of few, ascending, descending, in the period of the threads' pieces: equal ones by their index."""
    ramp = torch.arange(v, dtype=torch.float32)
    rows = [torch.zeros(v), torch.full((v,), -7.0), ramp / v * 8, -ramp / v * 8, ramp % 3, (ramp / 8).floor() % 2, (ramp % 4096 < 32) * 5.0, (ramp % 2048 < 8) * 5.0 - (ramp > 6000) * 1.0,
            torch.where(ramp % 2 == 0, 0.0, -0.0), (ramp % 1024 == 77) * 3.0, (ramp % 4096) / 512, (ramp >= v - 40) * 2.0 + (ramp == 3) * 2.0, (ramp % 384 < 24) * (ramp % 8) * 1.0,
            torch.where(ramp % 7 == 0, 1.0, -math.inf), torch.where(ramp > v - 30, 1.0, -math.inf)]
    logits = torch.stack(rows).to(dtype).to(cuda_device)
    tokens = torch.arange(len(rows), device=cuda_device) * 17
    for top in (1, 20, 32):
        check(logits, tokens, top)


@pytest.mark.parametrize("dtype", (F16, BF16, F32))
@pytest.mark.parametrize("vocab", (6, 301, 20000))
def test_masks_and_special_numbers(cuda_device, dtype, vocab):
    inf, nan = math.inf, math.nan
    low = torch.finfo(dtype).min
    base = logits_of(14, vocab, dtype, 9, "cpu")
    base[0] = -inf                                      # nothing may follow
    base[1] = -inf; base[1, vocab // 2] = 1.5           # one token only
    base[2] = -inf; base[2, ::3] = 0.25                 # a third, all alike
    base[3] = low                                       # all at the type's lowest
    base[4] = low; base[4, 1] = 2.0
    base[5, 0] = nan
    base[6, vocab - 1] = inf
    base[7] = nan
    base[8, 2] = inf; base[8, 3] = inf; base[8, 4] = nan
    base[9] = -inf; base[9, 0] = nan
    base[10, 1:] = -inf
    base[11] = -inf; base[11, -3:] = torch.tensor([1.0, 2.0, 1.0], dtype=dtype)
    base[12] = torch.finfo(dtype).max                   # finite, all alike
    logits = base.to(cuda_device)
    tokens = torch.tensor([0, vocab // 2, 1, 3, 0, 0, 0, 0, 3, 0, 0, vocab - 2, 5, -1], device=cuda_device)
    for top in (0, 3, min(32, vocab)):
        check(logits, tokens, top, 0.5 if top == 3 else 1.0)


def test_tokens_outside(cuda_device):
    logits = logits_of(6, 100, F16, 4, cuda_device)
    tokens = torch.tensor([-1, 99, 100, -(2 ** 40), 2 ** 40, 0], device=cuda_device)
    check(logits, tokens, 2)
    got = ab.token_logprobs(logits, tokens)
    assert got.logprobs[0] == 0 and got.logprobs[3] == 0 and bool(got.logprobs[[2, 4]].isnan().all()) and got.top_tokens.shape == (6, 0)


def test_strides(cuda_device):
    wide = logits_of(8, 2011, BF16, 5, cuda_device).view(2, 4, 2011)
    for logits in (wide, wide[..., :999], wide[..., 3:1001], wide[:, 1], wide.transpose(0, 1), wide[..., ::2], wide[1:, ::2, 5:2010], wide[:1, :1].expand(3, 2, 2011), wide[0, 0]):
        tokens = torch.randint(0, logits.shape[-1], logits.shape[:-1], generator=torch.Generator().manual_seed(2)).to(cuda_device)
        check(logits, tokens, 4)
    check(wide, torch.arange(16, device=cuda_device).view(2, 8)[:, ::2], 2)
    none = ab.token_logprobs(wide[:0], torch.zeros(0, 4, dtype=torch.int32, device=cuda_device), top=3)
    assert none.logprobs.shape == (0, 4) and none.top_tokens.shape == (0, 4, 3)


def test_many_rows_agree_with_few(cuda_device):
    """However many rows share a call, a row's answer is the same but for the order of its sums; its tokens are the same."""
    logits = logits_of(700, 5003, F16, 6, cuda_device)
    tokens = torch.randint(0, 5003, (700,), generator=torch.Generator().manual_seed(3)).to(cuda_device)
    many = ab.token_logprobs(logits, tokens, top=7)
    for r in (0, 1, 350, 699):
        one = ab.token_logprobs(logits[r:r + 1], tokens[r:r + 1], top=7)
        assert torch.equal(one.top_tokens, many.top_tokens[r:r + 1])
        for a, b in zip(one, many):
            assert torch.allclose(a.double(), b[r:r + 1].double(), rtol=1e-5, atol=1e-5)
    again = ab.token_logprobs(logits, tokens, top=7)
    assert all(torch.equal(a, b) for a, b in zip(many, again))


@pytest.mark.parametrize("dtype", (F16, BF16, F32))
@pytest.mark.parametrize("rows,vocab", [(1200, 5003), (800, 12289), (400, 20007)])
def test_many_long_rows(cuda_device, rows, vocab, dtype):
    """Rows of several batches a thread, with and without a rest, some of them masked in part or holding NaN."""
    logits = logits_of(rows, vocab, dtype, 10, cuda_device)
    logits[::7] = logits[::7].masked_fill(torch.rand(logits[::7].shape, generator=torch.Generator().manual_seed(4)).to(cuda_device) < 0.5, -math.inf)
    logits[3] = -math.inf
    logits[4, vocab - 2] = math.nan
    logits[5, : vocab // 2] = torch.finfo(dtype).min
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(5)).to(cuda_device)
    for top, temperature in ((0, 1.0), (12, 0.7)):
        check(logits, tokens, top, temperature)


def test_streams_and_graphs(cuda_device):
    logits, tokens = logits_of(3, 40000, BF16, 7, cuda_device), torch.tensor([1, 2, 3], device=cuda_device)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        ab.token_logprobs(logits, tokens, top=9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            found = ab.token_logprobs(logits, tokens, top=9)
            tokens.copy_(found.top_tokens[:, 0])   # the likeliest is the next to be asked for
    torch.cuda.synchronize(cuda_device)
    for seed in (8, 9):
        logits.copy_(logits_of(3, 40000, BF16, seed, cuda_device))
        graph.replay()
        graph.replay()
        torch.cuda.synchronize(cuda_device)
        assert torch.equal(found.logprobs, found.top_logprobs[:, 0])
        want = ab.token_logprobs(logits, tokens, top=9)
        assert torch.equal(want.top_tokens, found.top_tokens) and torch.equal(want.logprobs, found.logprobs)


def test_refusals(cuda_device):
    logits, tokens = torch.zeros(3, 50, dtype=F16, device=cuda_device), torch.zeros(3, dtype=torch.long, device=cuda_device)
    for bad, error in ((dict(logits=logits.double()), TypeError), (dict(logits=logits.cpu()), ValueError), (dict(tokens=tokens.float()), TypeError), (dict(tokens=tokens[:2]), ValueError),
                       (dict(tokens=tokens.cpu()), ValueError), (dict(top=-1), ValueError), (dict(top=51), ValueError), (dict(top=33), NotImplementedError),
                       (dict(temperature=0.0), ValueError), (dict(temperature=float("nan")), ValueError), (dict(temperature=-1.0), ValueError), (dict(logits=logits[:, :0]), ValueError),
                       (dict(temperature=float("inf")), ValueError)):
        with pytest.raises(error):
            ab.token_logprobs(**{"logits": logits, "tokens": tokens, **bad})
