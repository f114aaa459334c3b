"""The host side of the cache's operators: reports and refusals that need no GPU."""
import pytest
import torch

from atlasinfer_b200 import _capi, build
from atlasinfer_b200.integration import atlas_wrappers


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


def test_report_of_a_wait_that_ran_out():
    """The status word is shared by the linears and the attention: the report names both."""
    cpu = torch.device("cpu")
    atlas_wrappers.check_status(cpu)
    atlas_wrappers.status_word(cpu).fill_(1)
    with pytest.raises(_capi.AtlasError, match="attention") as e:
        atlas_wrappers.check_status(cpu)
    assert e.value.status == _capi.ERR_TIMEOUT
    atlas_wrappers.check_status(cpu)   # cleared


def test_index_types_are_checked(lib):
    """Positions and slots of neither 4 nor 8 bytes are refused, not read as 4.  (k is at no address that would be used.)"""
    for size in (0, 2, 16):
        t = _capi.Tokens(dtype=0, kv_heads=1, head_dim=64, tokens=1, k=17, k_out=16, table=16, positions=16, table_rows=4, rotary_dim=32, position_bytes=size)
        assert lib.atlas_norm_rotate(t, None) == _capi.ERR_BAD_ARGUMENT and b"positions" in lib.atlas_last_error()
        t = _capi.Tokens(dtype=0, kv_heads=1, head_dim=64, tokens=1, k=17, v=16, cache=16, num_pages=1, page_size=16, slots=16, slot_bytes=size)
        assert lib.atlas_norm_rotate(t, None) == _capi.ERR_BAD_ARGUMENT and b"slots" in lib.atlas_last_error()


@pytest.mark.parametrize("d,block", [(64, 256), (128, 256), (256, 128)])
def test_prompts_beyond_the_grid_are_refused(lib, d, block):
    """A sequence of more row blocks than a grid's second dimension holds: refused by name, not by a failed launch."""
    a = _capi.KvAttention(dtype=0, q_heads=64, kv_heads=1, head_dim=d, page_size=16, num_pages=1, max_pages=1, batch=1, q=17, out=16, cache=16, page_table=16, lengths=16)
    a.total_queries = a.max_queries = 65535 * block // 64 + 1
    assert lib.atlas_kv_attention(a, None) == _capi.ERR_UNSUPPORTED and b"queries in a sequence" in lib.atlas_last_error()
    a.total_queries = a.max_queries = 65535 * block // 64
    assert lib.atlas_kv_attention(a, None) == _capi.ERR_BAD_ARGUMENT   # (for its addresses, which are looked at after that)


def test_negative_bounds_are_refused():
    """max_queries below 0 is no way to say "all"."""
    import atlasinfer_b200 as ab

    for bad in (-1, -7):
        with pytest.raises(ValueError, match="max_queries"):
            ab.cache_attention(None, None, None, None, max_queries=bad)
