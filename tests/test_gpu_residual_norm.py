"""Norms with the residual sum against their definition in 64 bits."""
import pytest
import torch

import atlasinfer_b200 as ab

from . import decoder_reference as D
from .kv_reference import assert_rounded

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def randn(shape, dtype, seed, device, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


def check(got, stream, want, dtype):
    y, s, slack_y, slack_s = want
    assert got.dtype == dtype and got.is_contiguous()
    if stream.dtype == F32:
        assert bool(((stream.cpu().double() - s).abs() <= slack_s + s.abs() * 2.0 ** -24 + 2.0 ** -149).all())
    else:
        assert_rounded(stream, s, slack_s, "stream: ")
    assert_rounded(got, y, slack_y, "normed: ")


SHAPES = [(1, 1), (3, 7), (1, 4096), (5, 64), (2, 33), (17, 1000), (4, 8192), (2, 8200), (1, 16392), (2, 20001), (1, 32768), (700, 96), (3, 2049), (300, 2048), (2, 32767), (3, 32761), (1200, 33),
          (1300, 255), (1201, 257), (1190, 1013), (400, 4091), (300, 8181), (350, 10001), (310, 8200), (297, 1024)]


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("tokens,hidden", SHAPES)
def test_plain_norm(cuda_device, tokens, hidden, dtype):
    x = randn((tokens, hidden), dtype, 0, cuda_device, 3) + 0.5
    w, b = randn((hidden,), dtype, 1, cuda_device), randn((hidden,), F32, 2, cuda_device)
    for how in (dict(), dict(weight=w), dict(weight=w, bias=b, centered=True, eps=1e-5), dict(weight=b, weight_offset=1.0)):
        y, s = ab.residual_norm(x, **how)
        assert s is x   # nothing to add: the stream is x
        want = D.residual_norm(x, **how)
        check(y, s, want, dtype)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("stream_type", ("same", "fp32"))
@pytest.mark.parametrize("tokens,hidden,gate,post,centered", [
    (1, 4096, None, False, False), (3, 515, "rows", True, True), (33, 1024, "channels", True, False), (2, 16384, "rows", False, True), (130, 264, "channels", False, False),
    (1, 1, "rows", True, False), (2, 32768, "channels", True, True), (5, 5001, None, True, False),
    (350, 1003, "rows", True, True), (301, 1003, "channels", True, False), (1300, 200, "rows", False, True), (1250, 999, "rows", True, False), (320, 9000, "rows", True, False),
    (600, 4096, None, True, False), (741, 2048, "rows", True, True)])
def test_with_everything(cuda_device, tokens, hidden, gate, post, centered, stream_type, dtype):
    x = randn((tokens, hidden), dtype, 0, cuda_device)
    residual = randn((tokens, hidden), dtype if stream_type == "same" else F32, 1, cuda_device, 4)
    how = dict(weight=randn((hidden,), dtype, 2, cuda_device), bias=randn((hidden,), dtype, 3, cuda_device) if centered else None, scale=0.7, eps=1e-5, centered=centered,
               weight_offset=1.0, post_weight=randn((hidden,), F32, 4, cuda_device) if post else None)
    if gate:
        how["gate"] = randn((tokens, hidden) if gate == "rows" else (hidden,), dtype if tokens % 2 else F32, 5, cuda_device)
    kept = residual.clone()
    y, s = ab.residual_norm(x, residual, **how)
    assert s.dtype == residual.dtype and s.shape == x.shape and torch.equal(residual, kept)
    check(y, s, D.residual_norm(x, residual, **how), dtype)
    y2, s2 = ab.residual_norm(x, residual, **how)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    # without a residual the stream is the block in x's dtype
    y, s = ab.residual_norm(x, **how)
    check(y, s, D.residual_norm(x, **how), dtype)
    assert s.dtype == dtype


def test_shapes_and_strides(cuda_device):
    """Leading dimensions, views of wider rows at odd addresses, transposed rows, rows in reverse order: the numbers count."""
    wide = randn((6, 4, 200), BF16, 0, cuda_device)
    w = randn((96,), BF16, 1, cuda_device)
    for x in (wide[..., :96], wide[..., 1:97], wide.reshape(-1)[1:1 + 24 * 96].view(6, 4, 96), wide[:, 1, 8:104], wide[::2, :, 100:196], wide.transpose(0, 1)[..., :96], wide[:, :, 0:192:2], wide[:1, :1, 3:99].expand(5, 2, 96)):
        res = torch.flip(x, [0]).float()
        y, s = ab.residual_norm(x, res, w)
        want = D.residual_norm(x.reshape(-1, 96), res.reshape(-1, 96), w)
        assert y.shape == s.shape == x.shape
        check(y.reshape(-1, 96), s.reshape(-1, 96), want, BF16)
        y2, s2 = ab.residual_norm(x, x, w[:], gate=x)
        check(y2.reshape(-1, 96), s2.reshape(-1, 96), D.residual_norm(x.reshape(-1, 96), x.reshape(-1, 96), w, gate=x.reshape(-1, 96)), BF16)
    for rows in (wide[:, 0, :96], wide[:, 0, 1:96]):   # one row as the residual or the input of all
        res = rows[:1].expand(6, rows.shape[1])
        check(*ab.residual_norm(rows, res, w[:rows.shape[1]]), D.residual_norm(rows, res, w[:rows.shape[1]]), BF16)
        check(*ab.residual_norm(res, rows, w[:rows.shape[1]]), D.residual_norm(res, rows, w[:rows.shape[1]]), BF16)
    one = wide[0, 0, :96]
    assert ab.residual_norm(one, one, w)[0].shape == (96,)
    none = wide[:0, :, :96]
    y, s = ab.residual_norm(none, none, w)
    assert y.shape == s.shape == (0, 4, 96)
    odd = randn((97,), BF16, 2, cuda_device)[1:]   # weights at an odd address
    check(*ab.residual_norm(wide[:, 0, :96], None, odd), D.residual_norm(wide[:, 0, :96], None, odd), BF16)


@pytest.mark.parametrize("hidden", (64, 1001, 2051))
@pytest.mark.parametrize("wide", (False, True))
def test_stream_in_place(cuda_device, hidden, wide):
    """Through the C entry the stream may take the residual's place: rows that share 16 bytes with their neighbours too."""
    from atlasinfer_b200 import _capi

    tokens = 400
    x, r = randn((tokens, hidden), F16, 0, cuda_device), randn((tokens, hidden), F32 if wide else F16, 1, cuda_device, 3)
    w = randn((hidden,), F16, 2, cuda_device)
    y, s = ab.residual_norm(x, r, w)
    out = torch.empty_like(x)
    a = _capi.ResidualNorm(dtype=0, wide=int(wide), scale=1.0, eps=1e-6, tokens=tokens, hidden=hidden, x=x.data_ptr(), residual=r.data_ptr(), x_stride=hidden, residual_stride=hidden,
                           weight=w.data_ptr(), normed=out.data_ptr(), stream_out=r.data_ptr())
    assert _capi.load().atlas_residual_norm(a, _capi.stream_ptr(cuda_device)) == 0
    torch.cuda.synchronize(cuda_device)
    assert torch.equal(out, y) and torch.equal(r, s)


def test_special_numbers(cuda_device):
    inf, nan = float("inf"), float("nan")
    x = torch.ones(6, 64, dtype=F16, device=cuda_device)
    x[1, 3], x[2, 5] = nan, inf
    x[3] = 0
    x[4] = 60000.0
    x[5] = 6e-8
    y, s = ab.residual_norm(x, x, scale=1.0, eps=1e-6)
    assert bool(y[1].isnan().all()) and bool(y[2, 5].isnan()) and not y[3].any()
    assert bool((s[4] == inf).all()) and bool((y[4] == 1).all())   # the stream overflows fp16; what is normed is not rounded to it
    want = D.residual_norm(x[5:], x[5:])
    assert_rounded(y[5:], want[0], want[2])
    y, _ = ab.residual_norm(x[3:4], None, eps=0.0)   # 0 * rsqrt(0)
    assert bool(y.isnan().all())


def test_streams_and_graphs(cuda_device):
    x, res = randn((40, 1024), BF16, 0, cuda_device), randn((40, 1024), F32, 1, cuda_device)
    w = randn((1024,), BF16, 2, cuda_device)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        ab.residual_norm(x, res, w)
        with torch.cuda.graph(graph, stream=side):
            h, s = ab.residual_norm(x, res, w)
            y, s = ab.residual_norm(h, s, w)
    torch.cuda.synchronize(cuda_device)
    for seed in (5, 6):
        x.copy_(randn((40, 1024), BF16, seed, cuda_device))
        graph.replay()
        h2, s2 = ab.residual_norm(x, res, w)
        y2, s2 = ab.residual_norm(h2, s2, w)
        torch.cuda.synchronize(cuda_device)
        assert torch.equal(y, y2) and torch.equal(s, s2)


def test_refusals(cuda_device):
    x = torch.zeros(3, 64, dtype=F16, device=cuda_device)
    for bad, error in ((dict(x=x.float()), TypeError), (dict(x=x.cpu()), ValueError), (dict(residual=x[:2]), ValueError), (dict(residual=x.bfloat16()), TypeError),
                       (dict(residual=x.double()), TypeError), (dict(weight=x[0, :63]), ValueError), (dict(weight=x), ValueError), (dict(weight=x[0].cpu()), ValueError),
                       (dict(gate=x[:1]), ValueError), (dict(bias=x[0].double()), TypeError), (dict(post_weight=x[0].bfloat16()), TypeError),
                       (dict(x=x[:, :0]), ValueError), (dict(residual=x.cpu()), ValueError)):
        with pytest.raises(error):
            ab.residual_norm(**{"x": x, **bad})
    with pytest.raises(NotImplementedError):
        ab.residual_norm(torch.zeros(1, 32769, dtype=F16, device=cuda_device))
