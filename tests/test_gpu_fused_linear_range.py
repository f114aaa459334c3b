"""bf16 activations beyond fp16's range in the linears with an epilogue: as the modules themselves take them."""
import math

import pytest
import torch

import atlasinfer_b200 as ab

from . import decoder_reference as D
from .kv_reference import assert_rounded
from .test_gpu_fused_linear import module, randn

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
LARGEST = 65280.0   # the largest bf16 number that fp16 holds; what lies above (65536 is the next) becomes 65504


def ways(x):
    """The rows as they are, rows that lie off 16 bytes, and rows apart: every way into the kernels."""
    m, k = x.shape
    odd, wide = torch.empty(m * k + 1, dtype=x.dtype, device=x.device), torch.zeros(m, k + 24, dtype=x.dtype, device=x.device)
    odd[1:] = x.flatten()
    wide[:, 8:k + 8] = x
    return x, odd[1:].view(m, k), wide[:, 8:k + 8]


@pytest.mark.parametrize("n,k,block", [(256, 512, 128), (129, 256, 32)])
@pytest.mark.parametrize("m", (1, 2, 5, 12, 24, 60, 100, 128, 300))
def test_beyond_fp16(cuda_device, m, n, k, block):
    (lin, w), (up, v) = (module(n, k, s, cuda_device, block) for s in (1, 2))
    inf, most = math.inf, torch.finfo(BF16).max
    x = randn((m, k), BF16, m, cuda_device)
    x[0, :7] = torch.tensor([inf, -inf, most, -most, 65536.0, -1e30, LARGEST], dtype=BF16)
    x[m - 1, k - 3:] = torch.tensor([-inf, 70000.0, inf], dtype=BF16)
    # the same rows as fp16 numbers (small ones lose the same bits)
    as_fp16 = x.float().clamp(-65504.0, 65504.0).half()
    residual = randn((m, n), BF16, m + 1, cuda_device)
    residual[0, 3] = inf
    for rows in ways(x):
        assert torch.equal(ab.linear_epilogue(lin, rows), lin(rows))
        y = ab.linear_epilogue(lin, rows, "silu", residual=residual, scale=0.5)
        want, slack = D.fused(as_fp16, [w], [lin.bias], "silu", residual, 0.5)
        assert y[0, 3] == inf
        y[0, 3], want[0, 3] = 0, 0
        slack[0, 3] = 0
        assert_rounded(y, want, slack)
        scale = 2.0 ** -16
        z = ab.gated_linear(lin, up, rows, None, scale=scale)
        want, slack = D.fused(as_fp16, [w, v], [lin.bias, up.bias], None, None, scale)
        assert_rounded(z, want, slack)
        assert bool(z.isfinite().all())


@pytest.mark.parametrize("m", (1, 2, 5, 12, 24, 100, 300))
def test_nan_stays(cuda_device, m):
    (lin, _), (up, _) = (module(64, 128, s, cuda_device) for s in (3, 4))
    x = randn((m, 128), BF16, m, cuda_device)
    clean = x.clone()
    x[m - 1, 77] = math.nan
    for rows in ways(x):
        for call in (lambda t: ab.linear_epilogue(lin, t, "gelu"), lambda t: ab.gated_linear(lin, up, t)):
            y = call(rows)
            assert bool(y[m - 1].isnan().all()) and torch.equal(y[:m - 1], call(clean)[:m - 1])
