"""A decoder step from the stream to the answer: the operators together, each against its definition on what it was given."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import atlasinfer_b200 as ab

from . import decoder_reference as D
from .kv_reference import assert_rounded
from .test_gpu_fused_linear import module, randn

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,stream_type", ((BF16, BF16), (F16, F32)))
@pytest.mark.parametrize("tokens", (1, 3, 20, 140))
def test_step(cuda_device, tokens, dtype, stream_type):
    """Captured once and replayed for other tokens: attention's output projection, norms, MLP, answer, next token."""
    hidden, inter, vocab = 256, 640, 1111
    (o, wo), (gate, wg), (up, wu), (down, wd) = (module(n, k, s, cuda_device, bias=s == 1) for s, (n, k) in
                                                 enumerate(((hidden, hidden), (inter, hidden), (inter, hidden), (hidden, inter)), 1))
    ab.fuse_linears([gate, up])
    n1, n2, post = (randn((hidden,), dtype, s, cuda_device) for s in (5, 6, 7))
    head = randn((vocab, hidden), dtype, 8, cuda_device, 0.1)
    a, x = randn((tokens, hidden), dtype, 0, cuda_device), randn((tokens, hidden), stream_type, 1, cuda_device, 2)
    asked = torch.arange(tokens, device=cuda_device)

    def step():
        h, s = ab.residual_norm(o(a), x, n1, post_weight=post, eps=1e-5)
        m = ab.gated_linear(gate, up, h, "gelu_tanh")
        d = ab.linear_epilogue(down, m, residual=h, scale=0.5)   # (a parallel path takes the normed rows along)
        f, t = ab.residual_norm(d, s, n2, eps=1e-5)
        logits = f @ head.T
        found = ab.token_logprobs(logits, asked, top=3)
        return o(a), h, s, m, d, f, t, logits, found

    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            p, h, s, m, d, f, t, logits, found = step()
    torch.cuda.synchronize(cuda_device)
    for seed in (20, 21):
        a.copy_(randn((tokens, hidden), dtype, seed, cuda_device))
        x.copy_(randn((tokens, hidden), stream_type, seed + 5, cuda_device, 2))
        graph.replay()
        torch.cuda.synchronize(cuda_device)
        want, slack = D.fused(a, [wo], [o.bias], None)
        assert_rounded(p, want, slack)
        y, st, slack_y, slack_s = D.residual_norm(p, x, n1, post_weight=post, eps=1e-5)
        assert_rounded(h, y, slack_y)
        assert bool(((s.cpu().double() - st).abs() <= slack_s + st.abs() * (2.0 ** -24 if stream_type is F32 else 2.0 ** -8) + 2.0 ** -25).all())
        want, slack = D.fused(h, [wg, wu], [None, None], "gelu_tanh")
        assert_rounded(m, want, slack)
        want, slack = D.fused(m, [wd], [None], None, h, 0.5)
        assert_rounded(d, want, slack)
        y, _, slack_y, _ = D.residual_norm(d, s, n2, eps=1e-5)
        assert_rounded(f, y, slack_y)
        lp, ent, order, tops = D.token_logprobs(logits, asked, 3)
        assert torch.equal(found.top_tokens.cpu(), order)
        assert bool(((found.logprobs.cpu().double() - lp).abs() <= D.logprob_slack(vocab, lp, 1.0)).all())
        assert bool(((found.entropy.cpu().double() - ent).abs() <= 3 * (1 + ent) * D.logprob_slack(vocab, ent, 1.0)).all())
        assert bool(((found.top_logprobs.cpu().double() - tops).abs() <= D.logprob_slack(vocab, tops, 1.0)).all())


def test_first_calls_may_be_captured(cuda_device):
    """In a new process: nothing but the linears' layouts was there before the capture."""
    program = """
import torch
import atlasinfer_b200 as ab
gen = torch.Generator().manual_seed(3)
rand = lambda *s: torch.randn(*s, generator=gen).half().cuda()
up, down = (ab.QuantizedLinear(ab.quantize_tensor(rand(*s) * 0.05), None) for s in ((512, 256), (256, 512)))
up(rand(1, 256)), down(rand(1, 512))
for tokens in (1, 12, 30, 200):
    x = rand(tokens, 256)
    asked = torch.zeros(tokens, dtype=torch.long, device="cuda")

    def step():
        h, s = ab.residual_norm(x, x)
        y = ab.linear_epilogue(down, ab.gated_linear(up, up, h), "gelu", residual=s)
        return h, s, y, *ab.token_logprobs(y, asked, top=4)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step())), tokens
print("all of it")
"""
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0 and "all of it" in done.stdout, done.stderr[-2000:]


def test_calls_from_several_threads(cuda_device):
    """The operators on a stream of each thread's own, all with the same weights, at once."""
    (gate, _), (up, _), (down, _) = (module(n, k, s, cuda_device) for n, k, s in ((640, 256, 1), (640, 256, 2), (256, 640, 3)))
    norm = randn((256,), F16, 4, cuda_device)

    def step(x, asked):
        h, s = ab.residual_norm(x, x, norm)
        y = ab.linear_epilogue(down, ab.gated_linear(gate, up, h), residual=s)
        return (h, s, y, *ab.token_logprobs(y, asked, top=5))

    jobs = []
    for tokens in (1, 11, 40, 300):
        x, asked = randn((tokens, 256), F16, tokens, cuda_device), torch.arange(tokens, device=cuda_device) % 256
        jobs.append((x, asked, step(x, asked)))
    torch.cuda.synchronize(cuda_device)
    errors = []

    def work(x, asked, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream(cuda_device)):
                got = [step(x, asked) for _ in range(20)]
                torch.cuda.current_stream(cuda_device).synchronize()
                assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
        except BaseException as e:   # noqa: BLE001 - reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


def test_more_than_32_bits_of_numbers(cuda_device):
    """Tensors of more than 2^31 numbers: the last rows are as those of a small call's."""
    rows, hidden = 300000, 8192
    x = torch.empty(rows, hidden, dtype=BF16, device=cuda_device)
    x[-3:] = randn((3, hidden), BF16, 1, cuda_device)
    h, s = ab.residual_norm(x, x)
    y, st, slack, slack_s = D.residual_norm(x[-3:], x[-3:])
    assert_rounded(h[-3:], y, slack)
    assert_rounded(s[-3:], st, slack_s)
    del h, s
    wide = x.view(-1)[: 75001 * 32003].view(75001, 32003)
    wide[-2:] = randn((2, 32003), BF16, 2, cuda_device, 3)
    asked = torch.zeros(75001, dtype=torch.long, device=cuda_device)
    found = ab.token_logprobs(wide, asked, top=3)
    lp, _, order, _ = D.token_logprobs(wide[-2:], asked[-2:], 3)
    assert torch.equal(found.top_tokens[-2:].cpu(), order)
    assert bool(((found.logprobs[-2:].cpu().double() - lp).abs() <= D.logprob_slack(32003, lp, 1.0)).all())
    del wide, found
    (gate, wg), (up, wu) = (module(hidden, 256, s, cuda_device) for s in (3, 4))
    a = randn((rows, 256), BF16, 5, cuda_device)
    x[-3:] = randn((3, hidden), BF16, 6, cuda_device)
    got = ab.gated_linear(gate, up, a, residual=x)
    want, slack = D.fused(a[-3:], [wg, wu], [gate.bias, up.bias], "silu", x[-3:])
    assert_rounded(got[-3:], want, slack)
    got = ab.linear_epilogue(gate, a, "gelu", residual=x)
    want, slack = D.fused(a[-3:], [wg], [gate.bias], "gelu", x[-3:])
    assert_rounded(got[-3:], want, slack)
