"""What the cache's operators refuse, and what they need no GPU for."""
import ctypes

import pytest
import torch

import atlasinfer_b200 as ab
from atlasinfer_b200 import _capi, build

from . import kv_reference as R

F16 = torch.float16


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


def test_page_bytes(lib):
    for d in (64, 128, 256):
        for page in (16, 48, 64):
            assert lib.atlas_kv_page_bytes(d, page) == ab.QuantizedKVCache.page_bytes(d, page) == page * (d + 2 * d // 64 * 4)
    assert lib.atlas_kv_page_bytes(96, 16) == lib.atlas_kv_page_bytes(128, 24) == lib.atlas_kv_page_bytes(128, 0) == 0


def test_table():
    t = ab.rotary_table(100, 32, base=1000.0)
    assert t.shape == (100, 32) and t.dtype == torch.float32
    angle = 99 * 1000.0 ** (-6 / 32)
    assert abs(float(t[99, 3]) - torch.tensor(angle, dtype=torch.float64).cos()) < 1e-7 and abs(float(t[99, 19]) - torch.tensor(angle, dtype=torch.float64).sin()) < 1e-7
    with pytest.raises(ValueError):
        ab.rotary_table(10, 24)


def test_the_definition_itself():
    """Half a step at most, 15 steps for the range, zero exactly; 7 + 4 bits are exact in fp16."""
    x = torch.randn(50, 3, 128, generator=torch.Generator().manual_seed(0), dtype=torch.float64) * 7
    y, s = R.stored(x), R.steps(x)
    assert bool(((x - y).abs() <= s * (0.5 + 2.0 ** -6)).all()) and torch.equal(y.half().double(), y)
    z = torch.cat([x[..., :64], torch.zeros(50, 3, 64, dtype=torch.float64)], -1)
    assert not R.stored(z)[..., 64:].any()


def test_cache_refuses():
    for bad in (96, 32, 0, 512):
        with pytest.raises(NotImplementedError):
            ab.QuantizedKVCache(1, 1, bad)
    for bad in (0, 8, 24, -16, 1 << 21):
        with pytest.raises(NotImplementedError):
            ab.QuantizedKVCache(1, 1, 64, page_size=bad)
    with pytest.raises(ValueError):
        ab.QuantizedKVCache(1, 0, 64)
    with pytest.raises(ValueError):
        ab.QuantizedKVCache(-1, 1, 64)
    with pytest.raises(TypeError):
        ab.QuantizedKVCache(1, 1, 64, page_size=16, data=torch.zeros(1, 1, 1152))
    with pytest.raises(ValueError):
        ab.QuantizedKVCache(1, 1, 64, page_size=16, data=torch.zeros(1, 1, 1151, dtype=torch.uint8))
    with pytest.raises(ValueError):   # on the CPU
        ab.QuantizedKVCache(1, 1, 64, page_size=16, data=torch.zeros(1, 1, 1152, dtype=torch.uint8))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            ab.QuantizedKVCache(1, 1, 64)


def test_tensors_on_the_cpu_are_refused(lib):
    q, k = torch.zeros(2, 4, 64, dtype=F16), torch.zeros(2, 2, 64, dtype=F16)
    with pytest.raises(ValueError, match="CUDA"):
        ab.norm_rotate(q, k)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        ab.norm_rotate(q.float(), k.float())
    with pytest.raises(ValueError, match="tokens, heads, head_dim"):
        ab.norm_rotate(q, k[0])


def test_c_entries_check_before_cuda(lib):
    t = _capi.Tokens(dtype=0, q_heads=1, kv_heads=1, head_dim=80, tokens=1)
    assert lib.atlas_norm_rotate(t, None) == _capi.ERR_UNSUPPORTED and b"head_dim" in lib.atlas_last_error()
    t.head_dim, t.dtype = 64, 7
    assert lib.atlas_norm_rotate(t, None) == _capi.ERR_BAD_ARGUMENT
    t.dtype, t.tokens = 0, -1
    assert lib.atlas_norm_rotate(t, None) == _capi.ERR_BAD_ARGUMENT
    t.tokens = 0
    assert lib.atlas_norm_rotate(t, None) == _capi.OK
    t.tokens = 1
    t.k = t.k_out = t.q = t.q_out = 16
    t.table, t.positions, t.table_rows, t.rotary_dim = 16, 16, 4, 24
    assert lib.atlas_norm_rotate(t, None) == _capi.ERR_UNSUPPORTED and b"rotary_dim" in lib.atlas_last_error()
    assert lib.atlas_norm_rotate(None, None) == _capi.ERR_BAD_ARGUMENT
    assert lib.atlas_kv_load(None, 1, 1, 64, 16, None, 8, 1, 0, None, None, None) == _capi.ERR_BAD_ARGUMENT
    assert lib.atlas_kv_load(None, 1, 1, 64, 20, None, 8, 1, 0, None, None, None) == _capi.ERR_UNSUPPORTED
    a = _capi.KvAttention(dtype=0, q_heads=3, kv_heads=2, head_dim=64, page_size=16)
    assert lib.atlas_kv_attention(a, None) == _capi.ERR_BAD_ARGUMENT and b"query heads" in lib.atlas_last_error()
    a.q_heads, a.window = 4, -1
    assert lib.atlas_kv_attention(a, None) == _capi.ERR_BAD_ARGUMENT
    a.window, a.total_queries, a.batch = 0, 0, 0
    assert lib.atlas_kv_attention(a, None) == _capi.OK
    a.total_queries, a.batch, a.max_queries = 3, 2, 3
    assert lib.atlas_kv_attention(a, None) == _capi.ERR_BAD_ARGUMENT and b"query_starts" in lib.atlas_last_error()
    a.total_queries = 2
    a.q = a.out = a.lengths = 16
    a.workspace = 17
    assert lib.atlas_kv_attention(a, None) == _capi.ERR_BAD_ARGUMENT
    assert lib.atlas_kv_attention(None, None) == _capi.ERR_BAD_ARGUMENT
    assert ctypes.sizeof(_capi.Tokens) == 208 and ctypes.sizeof(_capi.KvAttention) == 168   # as in the header on this ABI


@pytest.mark.gpu
def test_refusals_on_the_gpu(cuda_device):
    z = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype, device=cuda_device)  # noqa: E731
    cache = ab.QuantizedKVCache(2, 2, 64, page_size=16, device=cuda_device)
    q, k, slots = z(3, 4, 64), z(3, 2, 64), z(3, dtype=torch.int64)
    table, positions = ab.rotary_table(8, 32, device=cuda_device), z(3, dtype=torch.int64)
    bad = [
        (TypeError, lambda: ab.norm_rotate(q.float(), k)), (TypeError, lambda: ab.norm_rotate(q.bfloat16(), k)), (ValueError, lambda: ab.norm_rotate(q[:2], k)),
        (ValueError, lambda: ab.norm_rotate(z(3, 4, 128), k)), (NotImplementedError, lambda: ab.norm_rotate(z(3, 4, 96), z(3, 2, 96))),
        (ValueError, lambda: ab.norm_rotate(q, k, table)), (ValueError, lambda: ab.norm_rotate(q, k, table, positions[:2])),
        (TypeError, lambda: ab.norm_rotate(q, k, table, positions.float())), (TypeError, lambda: ab.norm_rotate(q, k, table.half(), positions)),
        (NotImplementedError, lambda: ab.norm_rotate(q, k, z(8, 24, dtype=torch.float32), positions)),
        (NotImplementedError, lambda: ab.norm_rotate(q, k, z(8, 128, dtype=torch.float32), positions)),
        (ValueError, lambda: ab.norm_rotate(q, k, table, positions.cpu())), (ValueError, lambda: ab.norm_rotate(q, k, q_weight=z(32))),
        (TypeError, lambda: ab.norm_rotate(q, k, q_weight=z(64, dtype=torch.bfloat16))), (TypeError, lambda: ab.norm_rotate(q, k, q_weight=z(64), k_weight=z(64).float())),
        (ValueError, lambda: cache.store(k, z(3, 1, 64), slots)), (ValueError, lambda: cache.store(z(3, 1, 64), z(3, 1, 64), slots)),
        (ValueError, lambda: cache.store(z(3, 2, 128), z(3, 2, 128), slots)), (TypeError, lambda: cache.store(k, k.bfloat16(), slots)),
        (ValueError, lambda: cache.store(k, k, slots[:2])), (TypeError, lambda: cache.store(k, k, slots.float())),
        (TypeError, lambda: cache.load(slots, dtype=torch.float32)), (ValueError, lambda: cache.load(slots.cpu())),
    ]
    pages, lengths = z(3, 2, dtype=torch.int32), z(3, dtype=torch.int32)
    starts = z(4, dtype=torch.int32)
    attend = ab.cache_attention
    bad += [
        (TypeError, lambda: attend(q, cache, pages.long(), lengths)), (TypeError, lambda: attend(q, cache, pages, lengths.long())),
        (ValueError, lambda: attend(q, cache, pages[0], lengths)), (ValueError, lambda: attend(q, cache, pages, lengths[:2])),
        (ValueError, lambda: attend(z(3, 3, 64), cache, pages, lengths)), (ValueError, lambda: attend(z(3, 4, 128), cache, pages, lengths)),
        (TypeError, lambda: attend(q.float(), cache, pages, lengths)), (ValueError, lambda: attend(q[:2], cache, pages, lengths)),
        (ValueError, lambda: attend(q, cache, pages, lengths, query_starts=starts[:3])), (TypeError, lambda: attend(q, cache, pages, lengths, query_starts=starts.long())),
        (ValueError, lambda: attend(q, cache, pages, lengths, window=0)), (ValueError, lambda: attend(q, cache, pages, lengths, sinks=-1)),
        (ValueError, lambda: attend(q, cache, pages.cpu(), lengths)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print("not refused:", i)
    assert attend(q[:0], cache, pages[:0], lengths[:0]).shape == (0, 4, 64)
    assert ab.norm_rotate(q[:0], k[:0])[0].shape == (0, 4, 64)
    torch.cuda.synchronize()
