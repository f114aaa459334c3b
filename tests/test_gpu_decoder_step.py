"""A decoder step from the stream to the answer: the operators together, each against its definition on what it was given."""
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
