"""gated_linear where weights are large enough that other kernels take the few rows than those small weights go to."""
import ctypes

import pytest
import torch

import atlasinfer_b200 as ab
from atlasinfer_b200 import _capi

from . import decoder_reference as D
from .kv_reference import assert_rounded
from .test_gpu_fused_linear import module, randn

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def check_all(device, pair, weights, rows, dtype):
    """Every activation with and without a residual and a scale, the biases of both weights in each."""
    gate, up = pair
    n, k = weights[0].shape
    for m in rows:
        x, residual = randn((m, k), dtype, m, device), randn((m, n), dtype, m + 1, device)
        for i, act in enumerate(D.ACTIVATIONS):
            more, scale = (residual, -0.6) if i % 2 else (None, 1.0) if i % 3 else (residual, 1.0)
            y = ab.gated_linear(gate, up, x, act, residual=more, scale=scale)
            want, slack = D.fused(x, weights, [gate.bias, up.bias], act, more, scale)
            assert_rounded(y, want, slack, f"{n}x{k}, {m} rows, {act}: ")
            assert torch.equal(y, ab.gated_linear(gate, up, x, act, residual=more, scale=scale))


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("joined", (False, True))
@pytest.mark.parametrize("n,k,block", [(2368, 1024, 128), (2369, 1024, 128), (2500, 1088, 64), (2433, 2048, 32), (5121, 640, 128)])
def test_nine_to_sixteen_rows(cuda_device, n, k, block, joined, dtype):
    """On either side of 148 strips: pairs of CTAs up to there, tiles of 16 tokens from there on, ends of tiles of every kind."""
    (gate, w), (up, v) = (module(n, k, s, cuda_device, block) for s in (2, 3))
    if joined:
        ab.fuse_linears([gate, up])
    check_all(cuda_device, (gate, up), [w, v], (9, 12, 16), dtype)


@pytest.mark.parametrize("dtype", (F16, BF16))
def test_sixteen_rows_of_a_long_k(cuda_device, dtype):
    (gate, w), (up, v) = (module(2500, 8192, s, cuda_device) for s in (4, 5))
    check_all(cuda_device, (gate, up), [w, v], (9, 16), dtype)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("joined", (False, True))
def test_a_strip_of_either_weight_in_a_cta(cuda_device, joined, dtype):
    """Up to 8 rows of weights with more strips than run at once in pairs of CTAs; 4100 rows end 4 into the last strip."""
    (gate, w), (up, v) = (module(4100, 4096, s, cuda_device) for s in (6, 7))
    if joined:
        ab.fuse_linears([up, gate])
    check_all(cuda_device, (gate, up), [w, v], (1, 2, 3, 8), dtype)


@pytest.mark.parametrize("dtype", (F16, BF16))
def test_without_biases(cuda_device, dtype):
    """A bias of one weight only, in both kernels."""
    for n, k, rows in ((4100, 4096, (1, 8)), (2500, 1024, (9, 16))):
        (gate, w), (up, v) = (module(n, k, s, cuda_device, bias=s == 8) for s in (8, 9))
        for pair, weights in (((gate, up), [w, v]), ((up, gate), [v, w])):
            check_all(cuda_device, pair, weights, rows, dtype)


@pytest.mark.parametrize("dtype", (F16, BF16))
def test_epilogue_of_two_strips_in_a_cta(cuda_device, dtype):
    """One weight, two of its strips in a CTA: 257 pairs fill most of one wave, the last one has half a strip."""
    lin, w = module(8200, 4096, 10, cuda_device)
    for m in (1, 2, 3, 8):
        x, residual = randn((m, 4096), dtype, m, cuda_device), randn((m, 8200), dtype, m + 1, cuda_device)
        for i, act in enumerate(D.ACTIVATIONS):
            more, scale = (residual, 0.3) if i % 2 else (None, 1.0)
            want, slack = D.fused(x, [w], [lin.bias], act, more, scale)
            assert_rounded(ab.linear_epilogue(lin, x, act, residual=more, scale=scale), want, slack, f"{m} rows, {act}: ")
        assert torch.equal(ab.linear_epilogue(lin, x), lin(x))


def fused_there(x, weights, biases, act, residual, scale):
    """``decoder_reference.fused`` on the GPU."""
    bf16, xd = x.dtype is BF16, x.double()
    parts = []
    for w, b in zip(weights, biases):
        w, b = w.to(x.device).double(), b.double()
        y = xd @ w.T + b
        slack = (xd.abs() @ w.abs().T) * (w.shape[1] / 16 + 32) * 2 * D.U + (w.abs().sum(1) * 2.0 ** -25 if bf16 else 0)
        parts.append((y, slack + D.U * y.abs()))
    v, off = parts[0]
    y = D.ACTIVATIONS[act](v)
    off = 1.13 * off + y.abs() * (16 + 8 * v.abs().clamp(max=100)) * D.U + 2.0 ** -126
    for u, more in parts[1:]:
        y, off = y * u, off * u.abs() + y.abs() * more + off * more
    y, off = y * scale, (off + 2 * D.U * y.abs()) * abs(scale)
    if residual is not None:
        y = y + residual.double()
        off = off + D.U * y.abs()
    return y.cpu(), off.cpu()


# (token tile, whether K is sliced), rows of the weight, K, tokens
TWO_WEIGHTS = [((160, False), 700, 256, 129), ((160, True), 700, 2048, 129), ((192, False), 5000, 512, 175), ((192, True), 1003, 2048, 497), ((224, False), 5000, 256, 175),
               ((224, True), 2500, 2048, 198), ((256, False), 5000, 256, 244), ((256, True), 700, 2048, 175), ((320, False), 5000, 256, 267), ((320, True), 2047, 4096, 267),
               ((384, False), 5000, 256, 336), ((384, True), 2500, 4096, 336)]
ONE_WEIGHT = [((160, False), 700, 256, 129), ((160, True), 700, 1024, 129), ((192, False), 6001, 1024, 175), ((192, True), 3001, 2048, 336), ((224, False), 7001, 256, 336),
              ((224, True), 1500, 2048, 658), ((256, False), 5000, 256, 497), ((256, True), 1003, 2048, 175), ((320, False), 7001, 256, 520), ((320, True), 4100, 4096, 267),
              ((384, False), 7001, 256, 658), ((384, True), 5000, 4096, 336)]


@pytest.mark.parametrize("count,tile,n,k,m", [(2, *c) for c in TWO_WEIGHTS] + [(1, *c) for c in ONE_WEIGHT])
def test_every_prompt_tile(cuda_device, count, tile, n, k, m):
    """With and without slices of K; two weights take the tiles of one with twice as many rows (in halves of 64)."""
    tokens, slices = ctypes.c_int(), ctypes.c_int()
    _capi.check(_capi.load().atlas_qlinear_gemm_plan(m, n if count == 1 else -(-n // 64) * 128, k, ctypes.byref(tokens), ctypes.byref(slices)), "plan")
    assert (tokens.value, slices.value > 1) == tile
    mods, weights = zip(*(module(n, k, 11 + i, cuda_device) for i in range(count)))
    biases = [mod.bias for mod in mods]
    call = ab.linear_epilogue if count == 1 else ab.gated_linear
    for i, dtype in enumerate((F16, BF16)):
        x, residual = randn((m, k), dtype, m, cuda_device), randn((m, n), dtype, m + 1, cuda_device)
        for act, more, scale in ((None, residual, 0.5), ("gelu_tanh", None, 1.0), ("silu", residual, -0.6)):
            want, slack = fused_there(x, weights, biases, act, more, scale)
            assert_rounded(call(*mods, x, act, residual=more, scale=scale), want, slack, f"{dtype}, {act}: ")
