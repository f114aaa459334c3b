"""Norms with the residual sum on either side of every change of kernel, with rows that lie in every way."""
import pytest
import torch

import atlasinfer_b200 as ab

from . import decoder_reference as D
from .test_gpu_residual_norm import BF16, F16, F32, check, randn

pytestmark = pytest.mark.gpu


def calls(x, residuals, seed):
    """The operator with and without all there is, on each residual."""
    device, hidden, dtype = x.device, x.shape[1], x.dtype
    w, b, post = randn((hidden,), dtype, seed, device), randn((hidden,), dtype, seed + 1, device), randn((hidden,), F32, seed + 2, device)
    gate = randn(tuple(x.shape), dtype, seed + 3, device)
    for residual in residuals:
        yield residual, dict(weight=w)
        yield residual, dict(weight=w, bias=b, post_weight=post, gate=gate, scale=0.7, eps=1e-5, centered=True, weight_offset=1.0)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("tokens,hidden", [(4096, 528), (4100, 768), (4097, 761), (4095, 768), (4096, 776), (1184, 512), (1184, 520), (1183, 264), (1184, 505)])
def test_short_rows(cuda_device, tokens, hidden, dtype):
    """A warp a row, or a CTA: 512 numbers, 768 of many rows with a stream of 16 bits; rows apart take numbers one by one."""
    wide = randn((tokens, hidden + 3), dtype, 0, cuda_device, 2)
    same, apart = randn((tokens, hidden), dtype, 1, cuda_device, 3), randn((tokens, hidden), F32, 2, cuda_device, 3)
    for x in (randn((tokens, hidden), dtype, 3, cuda_device) + 0.5, wide[:, 1:hidden + 1]):
        for residual, how in calls(x, (None, same, apart), 4):
            check(*ab.residual_norm(x, residual, **how), D.residual_norm(x, residual, **how), dtype)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("hidden,edge", [(4096, 592), (4096, 740), (5001, 444), (5001, 592), (4600, 444), (3500, 592), (5128, 592), (2048, 296)])
def test_a_few_hundred_rows(cuda_device, hidden, edge, dtype):
    """Rows that just fit at once in CTAs of many or of few registers, and one row more: the same numbers, bit for bit."""
    x = randn((edge + 1, hidden), dtype, 0, cuda_device) + 0.25
    same, apart = randn((edge + 1, hidden), dtype, 1, cuda_device, 3), randn((edge + 1, hidden), F32, 2, cuda_device, 3)
    for residual, how in calls(x, (same, apart), 4):
        more = ab.residual_norm(x, residual, **how)
        check(*more, D.residual_norm(x, residual, **how), dtype)
        how = {k: v[:edge] if k == "gate" else v for k, v in how.items()}
        fewer = ab.residual_norm(x[:edge], residual[:edge], **how)
        if edge != 296:   # (up to there a row has twice the threads)
            assert torch.equal(fewer[0], more[0][:edge]) and torch.equal(fewer[1], more[1][:edge])
        check(*fewer, D.residual_norm(x[:edge], residual[:edge], **how), dtype)
