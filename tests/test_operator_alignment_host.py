"""Buffers that lie off their types' or copies' boundaries are refused on the host.  (Addresses are never used.)"""
import pytest

from atlasinfer_b200 import _capi

from .test_decoder_ops_host import lib, linear, logprobs  # noqa: F401

FINE = dict(tiles=16, scales_tiled=16, outlier_chunk_ptr=16)
OFF = (dict(tiles=24), dict(scales_tiled=24), dict(scales_tiled=18), dict(outlier_chunk_ptr=18), dict(outlier_entries=18), dict(outlier_vals_sorted=17), dict(bias=17))


@pytest.mark.parametrize("m", (1, 4, 12, 40, 400))
@pytest.mark.parametrize("off", OFF)
def test_weights(lib, m, off):  # noqa: F811
    bad = _capi.Weight(**{**FINE, **off})
    for a in (linear(m, weight=bad), linear(m, up=bad), linear(m, up=True, weight=bad)):
        assert lib.atlas_fused_linear(a, None) == _capi.ERR_BAD_ARGUMENT and b"aligned" in lib.atlas_last_error()


@pytest.mark.parametrize("m,up", [(m, up) for m in (1, 4, 40, 400) for up in (False, True)])
@pytest.mark.parametrize("off", (dict(x=17), dict(y=17), dict(residual=17, ldr=64), dict(residual=16 + 1, ldr=65), dict(status=18)))
def test_rows(lib, m, up, off):  # noqa: F811
    assert lib.atlas_fused_linear(linear(m, up, **off), None) == _capi.ERR_BAD_ARGUMENT and b"aligned" in lib.atlas_last_error()


@pytest.mark.parametrize("off", (dict(logprobs=18), dict(entropy=18), dict(top_logprobs=18), dict(top_tokens=20), dict(logits=17), dict(tokens=18, token_bytes=4)))
def test_log_probabilities(lib, off):  # noqa: F811
    assert lib.atlas_token_logprobs(logprobs(**off), None) == _capi.ERR_BAD_ARGUMENT and b"aligned" in lib.atlas_last_error()


def test_scales_of_plain_linears(lib):  # noqa: F811
    def call(scales, block):
        return lib.atlas_qlinear_gemm(16, 0, 40, 128, 16, scales, 16, None, None, 64, 128, block, None, 16, 64, 256, 1 << 40, None, None)

    for block in (64, 128):   # copied in 16-byte units
        assert call(18, block) == call(24, block) == _capi.ERR_BAD_ARGUMENT and b"scales_tiled" in lib.atlas_last_error()
