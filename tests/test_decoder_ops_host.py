"""The host side of the operators around a decoder step's linears: refusals that need no GPU.  (Addresses are never used.)"""
import ctypes
import math

import pytest
import torch

import atlasinfer_b200 as ab
from atlasinfer_b200 import _capi, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


def norm(**how):
    return _capi.ResidualNorm(**{**dict(dtype=0, tokens=2, hidden=64, x=16, normed=16, scale=1.0, eps=1e-6, x_stride=64), **how})


@pytest.mark.parametrize("how,status", [
    (dict(dtype=2), 1), (dict(dtype=-1), 1), (dict(hidden=0), 1), (dict(tokens=-1), 1), (dict(hidden=32769), 2), (dict(tokens=1 << 31), 2), (dict(x=None), 1), (dict(normed=None), 1),
    (dict(x=17), 1), (dict(weight=18, wide=4), 1), (dict(residual=18, wide=1), 1), (dict(gate=17), 1), (dict(bias=18, wide=8), 1), (dict(post_weight=18, wide=16), 1)])
def test_residual_norm_is_checked(lib, how, status):
    assert lib.atlas_residual_norm(norm(**how), None) == status and b"atlas_residual_norm" in lib.atlas_last_error()


def test_nothing_to_do(lib):
    assert lib.atlas_residual_norm(norm(tokens=0, x=None, normed=None), None) == 0
    assert lib.atlas_token_logprobs(logprobs(rows=0, logits=None), None) == 0
    assert lib.atlas_fused_linear(linear(m=0, x=None), None) == 0
    for name in ("atlas_residual_norm", "atlas_token_logprobs", "atlas_fused_linear"):
        assert getattr(lib, name)(None, None) == _capi.ERR_BAD_ARGUMENT


def logprobs(**how):
    return _capi.TokenLogprobs(**{**dict(dtype=0, top=2, token_bytes=8, temperature=1.0, rows=2, vocab=100, logits_stride=100, logits=16, tokens=16, logprobs=16, entropy=16, top_tokens=16,
                                         top_logprobs=16), **how})


@pytest.mark.parametrize("how,status", [
    (dict(dtype=3), 1), (dict(rows=-1), 1), (dict(vocab=0), 1), (dict(rows=1 << 31), 2), (dict(vocab=(1 << 30) + 1), 2), (dict(top=-1), 1), (dict(top=101), 1), (dict(top=33), 2),
    (dict(temperature=0.0), 1), (dict(temperature=-1.0), 1), (dict(temperature=math.nan), 1), (dict(temperature=math.inf), 1), (dict(token_bytes=2), 1), (dict(logits=None), 1),
    (dict(tokens=None), 1), (dict(logprobs=None), 1), (dict(entropy=None), 1), (dict(top_tokens=None), 1), (dict(top_logprobs=None), 1), (dict(logits=17), 1), (dict(logits=18, dtype=2), 1),
    (dict(tokens=20), 1)])
def test_token_logprobs_is_checked(lib, how, status):
    assert lib.atlas_token_logprobs(logprobs(**how), None) == status and b"atlas_token_logprobs" in lib.atlas_last_error()


def linear(m=4, up=False, weight=None, **how):
    w = _capi.Weight(tiles=16, scales_tiled=16, outlier_chunk_ptr=16)
    a = _capi.FusedLinear(**{**dict(dtype=0, activation=1, x=16, m=m, ldx=128, n_rows=64, n_cols=128, block_size=128, scale=1.0, weight=weight or w, y=16, ldy=64, workspace=256,
                                    workspace_bytes=1 << 40), **how})
    if up:
        a.up = up if isinstance(up, _capi.Weight) else w
    return a


@pytest.mark.parametrize("m,up", [(4, False), (40, False), (400, False), (4, True), (40, True), (400, True)])
@pytest.mark.parametrize("how,status", [
    (dict(activation=5), 1), (dict(activation=-1), 1), (dict(m=-1), 1), (dict(n_rows=0), 1), (dict(n_cols=0), 1), (dict(dtype=2), 1), (dict(residual=16, ldr=63), 1), (dict(x=None), 1),
    (dict(y=None), 1), (dict(n_cols=100, ldx=100), 2), (dict(block_size=48), 2), (dict(ldx=127), 1), (dict(ldy=63), 1), (dict(weight=_capi.Weight(tiles=16, scales_tiled=16)), 1)])
def test_fused_linear_is_checked(lib, m, up, how, status):
    assert lib.atlas_fused_linear(linear(**{"m": m, "up": up, **how}), None) == status and lib.atlas_last_error()


@pytest.mark.parametrize("m", (4, 40, 400))
def test_second_weights_and_workspaces(lib, m):
    for bad in (_capi.Weight(tiles=16, scales_tiled=16), _capi.Weight(tiles=16, outlier_chunk_ptr=16), _capi.Weight(tiles=24, scales_tiled=16, outlier_chunk_ptr=16)):
        assert lib.atlas_fused_linear(linear(m, bad), None) == _capi.ERR_BAD_ARGUMENT
    need = lib.atlas_fused_linear_workspace_bytes(linear(m, True))
    one = lib.atlas_fused_linear_workspace_bytes(linear(m))
    assert (one == 0) == (m <= 16)
    if need:
        assert lib.atlas_fused_linear(linear(m, True, workspace_bytes=need - 1), None) == _capi.ERR_CAPACITY
        assert lib.atlas_fused_linear(linear(m, True, workspace=264), None) == _capi.ERR_BAD_ARGUMENT
    assert lib.atlas_fused_linear_workspace_bytes(None) == 0
    assert lib.atlas_fused_linear_workspace_bytes(linear(m, activation=9)) == 0


def test_structs_have_the_header_s_sizes():
    """(on a 64-bit machine; the fields are read by name in the tests above)"""
    assert ctypes.sizeof(_capi.Weight) == 48
    assert ctypes.sizeof(_capi.FusedLinear) == 8 + 8 + 32 + 8 + 96 + 16 + 16 + 16 + 8
    assert ctypes.sizeof(_capi.ResidualNorm) == 24 + 16 + 24 + 24 + 24 + 16
    assert ctypes.sizeof(_capi.TokenLogprobs) == 16 + 24 + 16 + 16 + 16


def test_python_refusals():
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="activation"):
        ab.linear_epilogue(None, x, "swish")
    with pytest.raises(ValueError, match="CUDA"):
        ab.gated_linear(None, None, x)
    for t in (0, -1, math.nan, math.inf, 1e5, 1e-5):
        with pytest.raises(ValueError, match="temperature"):
            ab.token_logprobs(x, x, temperature=t)
    with pytest.raises(ValueError, match="CUDA"):
        ab.residual_norm(x)
    with pytest.raises(TypeError):
        ab.residual_norm(x.double())
    with pytest.raises(ValueError, match="CUDA"):
        ab.token_logprobs(x, torch.zeros(2, dtype=torch.long))
    with pytest.raises(TypeError):
        ab.token_logprobs(x.double(), torch.zeros(2, dtype=torch.long))
