"""Quantized linears with an epilogue against their definition in 64 bits."""
import pytest
import torch

import atlasinfer_b200 as ab

from . import decoder_reference as D
from .kv_reference import assert_rounded
from .util import config_weights

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def randn(shape, dtype, seed, device, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


def module(n, k, seed, device, block=128, bias=True):
    q = ab.quantize_tensor(config_weights(n, k, seed).to(device), block_size=block)
    w = ab.dequantize_tensor(q, device).cpu()
    ab.clear_dequantized_cache()
    b = randn((n,), F16, seed + 50, device, 0.2) if bias else None
    return ab.QuantizedLinear(q, b), w


# rows of x: every kernel, its token tiles and their edges; the weight: whole and ragged tiles, short and long K, small blocks
ROWS = (1, 2, 3, 8, 9, 16, 17, 33, 64, 65, 100, 128, 129, 300, 513)
WEIGHTS = [(256, 512, 128), (100, 64, 64), (1000, 1024, 32), (384, 4096, 128), (129, 192, 64), (64, 320, 16), (37, 1280, 256)]


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("n,k,block", WEIGHTS)
def test_epilogue(cuda_device, n, k, block, dtype):
    if block % 32:
        lin, w = module(n, k, 1, cuda_device, 64)
        lin = ab.QuantizedLinear(split_blocks(lin.quantized_weights, block), lin.bias)
    else:
        lin, w = module(n, k, 1, cuda_device, block)
    for i, m in enumerate(ROWS):
        x = randn((m, k), dtype, m, cuda_device)
        act = list(D.ACTIVATIONS)[i % 5]
        residual = randn((m, n), dtype, m + 1, cuda_device) if i % 3 else None
        scale = 1.0 if i % 2 else 0.3
        y = ab.linear_epilogue(lin, x, act, residual=residual, scale=scale)
        want, slack = D.fused(x, [w], [lin.bias], act, residual, scale)
        assert y.shape == (m, n) and y.dtype == dtype
        assert_rounded(y, want, slack, f"{m} rows, {act}: ")
        # without anything behind it, the linear itself, bit for bit
        assert torch.equal(ab.linear_epilogue(lin, x), lin(x))


def split_blocks(q, block):
    """The same weight in smaller blocks (of the same scales)."""
    times = q.block_size // block
    return ab.QuantizedTensor(q.fp8_data, q.fp16_outliers, q.outlier_indices, q.scale_factors.repeat_interleave(times), q.original_shape, block)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("joined", (False, True))
@pytest.mark.parametrize("n,k,block", WEIGHTS)
def test_gated(cuda_device, n, k, block, joined, dtype):
    bias = n != 1000
    size = block if block % 32 == 0 else 64
    (gate, w), (up, v) = (module(n, k, s, cuda_device, size, bias) for s in (2, 3))
    if size != block:
        gate, up = (ab.QuantizedLinear(split_blocks(m.quantized_weights, block), m.bias) for m in (gate, up))
    if joined:
        ab.fuse_linears([up, gate])   # (in whichever order)
    for i, m in enumerate(ROWS):
        x = randn((m, k), dtype, m, cuda_device)
        act = list(D.ACTIVATIONS)[(i + 2) % 5]
        residual = randn((m, n), dtype, m + 1, cuda_device) if i % 4 == 1 else None
        scale = 1.0 if i % 3 else -0.6
        y = ab.gated_linear(gate, up, x, act, residual=residual, scale=scale)
        want, slack = D.fused(x, [w, v], [gate.bias, up.bias], act, residual, scale)
        assert_rounded(y, want, slack, f"{m} rows, {act}: ")
        assert torch.equal(y, ab.gated_linear(gate, up, x, act, residual=residual, scale=scale))


def test_large(cuda_device):
    """More tiles than SMs, K slices in clusters, prompts of several token tiles."""
    for n, k, rows in ((11008, 4096, (1, 8, 32)), (4096, 11008, (1, 32, 200)), (4096, 4096, (1, 5, 48, 700)), (2048, 8192, (40, 128, 300))):
        (gate, w), (up, v) = (module(n, k, s, cuda_device, bias=False) for s in (2, 3))
        ab.fuse_linears([gate, up])
        wd, vd = w.to(cuda_device).double(), v.to(cuda_device).double()
        for m in rows:
            x, residual = randn((m, k), BF16, m, cuda_device), randn((m, n), BF16, m + 1, cuda_device)
            xd = x.double()
            g, u = xd @ wd.T, xd @ vd.T
            mass_g, mass_u = xd.abs() @ wd.abs().T, xd.abs() @ vd.abs().T
            c = (k / 16 + 32) * 2 * D.U
            off_g, off_u = mass_g * c + wd.abs().sum(1) * 2.0 ** -25, mass_u * c + vd.abs().sum(1) * 2.0 ** -25
            want = g * torch.sigmoid(g)
            off = (1.13 * off_g + want.abs() * (16 + 8 * g.abs()) * D.U) * (u.abs() + off_u) + want.abs() * off_u + 4 * D.U * (want * u).abs()
            assert_rounded(ab.gated_linear(gate, up, x), (want * u).cpu(), off.cpu(), f"gated {n}x{k}, {m} rows: ")
            want, off = residual.double() + 0.5 * g, 0.5 * off_g + D.U * (residual.double().abs() + g.abs())
            assert_rounded(ab.linear_epilogue(gate, x, residual=residual, scale=0.5), want.cpu(), off.cpu(), f"residual {n}x{k}, {m} rows: ")


def test_shapes_and_strides(cuda_device):
    (gate, w), (up, v) = (module(200, 256, s, cuda_device) for s in (4, 5))
    wide = randn((5, 7, 600), F16, 0, cuda_device)
    far = randn((5, 7, 700), F16, 1, cuda_device)
    for m in (1, 2, 5):
        for x in (wide[:m, :, :256], wide[:m, :, 3:259], wide[:m, 2, 8:264], wide[:m, :3].transpose(0, 1)[..., :256], wide[:m, :, 0:512:2], wide[:1, 0, :256].expand(m, 256)):
            residual = far[..., :200].expand(5, 7, 200)[:x.shape[0], :x.shape[1]] if x.dim() == 3 and x.shape[0] <= 5 and x.shape[1] <= 7 else far[:x.shape[0], 0, 1:201]
            for y, ws, bs in ((ab.linear_epilogue(gate, x, "silu", residual=residual), [w], [gate.bias]),
                              (ab.gated_linear(gate, up, x, "silu", residual=residual), [w, v], [gate.bias, up.bias])):
                want, slack = D.fused(x.reshape(-1, 256), ws, bs, "silu", residual.reshape(-1, 200))
                assert y.shape == (*x.shape[:-1], 200)
                assert_rounded(y.reshape(-1, 200), want, slack)
    assert ab.gated_linear(gate, up, wide[:0, 0, :256]).shape == (0, 200)
    assert ab.linear_epilogue(gate, wide[0, 0, :256], "relu").shape == (200,)


def test_special_numbers(cuda_device):
    """Products that overflow, activations far out, NaN in a row: as the formula has them; other rows keep their bits."""
    lin, w = module(128, 128, 6, cuda_device, bias=False)
    up, v = module(128, 128, 7, cuda_device, bias=False)
    for m in (4, 40, 200):
        x = randn((m, 128), F16, 8, cuda_device)
        x[1] *= 100
        clean = x.clone()
        x[2, 5] = float("nan")
        for act in D.ACTIVATIONS:
            for call in (lambda t: ab.linear_epilogue(lin, t, act), lambda t: ab.gated_linear(lin, up, t, act)):
                y, z = call(x), call(clean)
                assert bool(y[2].isnan().all())
                keep = [i for i in range(m) if i != 2]
                assert torch.equal(y[keep], z[keep]) and bool(z.isfinite().all())
            want, slack = D.fused(clean[:2], [w], [None], act)
            assert_rounded(ab.linear_epilogue(lin, clean, act)[:2], want, slack)


def test_streams_graphs_and_first_use(cuda_device):
    """Weights that are laid out by the call itself; captured and replayed on other inputs; two graphs on two streams."""
    (gate, w), (up, v), (down, d) = (module(n, k, s, cuda_device, bias=False) for n, k, s in ((512, 256, 8), (512, 256, 9), (256, 512, 10)))

    def mlp(t):
        return ab.linear_epilogue(down, ab.gated_linear(gate, up, t), residual=t)

    for m in (1, 20, 150):
        x = randn((m, 256), BF16, m, cuda_device)
        first = mlp(x)   # (the first time, behind the layouts' own kernels)
        graphs, outs, ins = [], [], []
        for i in range(2):
            s = torch.cuda.Stream(cuda_device)
            s.wait_stream(torch.cuda.current_stream(cuda_device))
            ins.append(x.clone())
            with torch.cuda.stream(s):
                mlp(ins[i])
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    outs.append(mlp(ins[i]))
                graphs.append((g, s))
        torch.cuda.synchronize(cuda_device)
        for i, (g, s) in enumerate(graphs):
            ins[i].copy_(randn((m, 256), BF16, 60 + i, cuda_device))
        torch.cuda.synchronize(cuda_device)
        for _ in range(3):
            for g, s in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize(cuda_device)
        for i in range(2):
            assert torch.equal(outs[i], mlp(ins[i]))
        assert torch.equal(first, mlp(x))


@pytest.mark.parametrize("m", (1, 5, 12, 40, 140))
def test_shared_tensors(cuda_device, m):
    """One module as gate and as up, the input as the residual, members of a group of three, calls on two streams at once."""
    (a, w), (b, v), (c, u) = (module(256, 256, s, cuda_device) for s in (12, 13, 14))
    x = randn((m, 256), F16, m, cuda_device)
    want, slack = D.fused(x, [w, w], [a.bias, a.bias], "gelu", x, 0.5)
    assert_rounded(ab.gated_linear(a, a, x, "gelu", residual=x, scale=0.5), want, slack)
    ab.fuse_linears([a, b, c])
    want, slack = D.fused(x, [u, v], [c.bias, b.bias], "silu")
    assert_rounded(ab.gated_linear(c, b, x), want, slack)
    assert_rounded(c(x), *D.fused(x, [u], [c.bias], None))
    torch.cuda.synchronize(cuda_device)
    streams, outs = [torch.cuda.Stream(cuda_device) for _ in range(2)], []
    inputs = [x, randn((m, 256), F16, m + 1, cuda_device)]
    torch.cuda.synchronize(cuda_device)
    for _ in range(5):
        for s, t in zip(streams, inputs):
            with torch.cuda.stream(s):
                outs.append(ab.linear_epilogue(a, ab.gated_linear(b, c, t), "relu", residual=t))
    torch.cuda.synchronize(cuda_device)
    for i, t in enumerate(inputs):
        want = ab.linear_epilogue(a, ab.gated_linear(b, c, t), "relu", residual=t)
        assert all(torch.equal(o, want) for o in outs[i::2])


def test_modules_and_refusals(cuda_device):
    (gate, w), (up, v), (small, _) = (module(n, 256, s, cuda_device) for n, s in ((64, 1), (64, 2), (32, 3)))
    x = torch.zeros(3, 256, dtype=F16, device=cuda_device)
    y = torch.zeros(3, 64, dtype=F16, device=cuda_device)
    for bad, error in ((lambda: ab.linear_epilogue(gate, x.float()), TypeError), (lambda: ab.linear_epilogue(gate, x[:, :255]), ValueError),
                       (lambda: ab.linear_epilogue(gate, x.cpu()), ValueError), (lambda: ab.linear_epilogue(gate, x, "tanh"), ValueError),
                       (lambda: ab.linear_epilogue(gate, x, residual=y[:2]), ValueError), (lambda: ab.linear_epilogue(gate, x, residual=y.bfloat16()), TypeError),
                       (lambda: ab.linear_epilogue(torch.nn.Linear(256, 64), x), TypeError), (lambda: ab.gated_linear(gate, small, x), ValueError),
                       (lambda: ab.linear_epilogue(gate, x, residual=y.cpu()), ValueError)):
        with pytest.raises(error):
            bad()
    # a module whose weight is given anew, grouped or not, computes with the new one
    x = randn((3, 256), F16, 4, cuda_device)
    ab.fuse_linears([gate, up])
    before = ab.gated_linear(gate, up, x)
    other, u = module(64, 256, 11, cuda_device)
    up.quantized_weights = other.quantized_weights
    want, slack = D.fused(x, [w, u], [gate.bias, up.bias], "silu")
    assert_rounded(ab.gated_linear(gate, up, x), want, slack)
    want, slack = D.fused(x, [w, v], [gate.bias, up.bias], "silu")
    assert_rounded(before, want, slack)
    # kept on the host, moved when needed; fp32 biases; only the layout on the GPU
    host = ab.QuantizedLinear(other.quantized_weights.to(torch.device("cpu")), up.bias.float().cpu())
    want, slack = D.fused(x, [u], [up.bias], "gelu")
    assert_rounded(ab.linear_epilogue(host, x, "gelu"), want, slack)
    host.offload_canonical()
    assert_rounded(ab.linear_epilogue(host, x, "gelu"), want, slack)
