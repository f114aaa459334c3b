"""Attention over the 4-bit cache at the edges: of numbers, of sequences, of the memory around what is seen."""
import pytest
import torch

import atlasinfer_b200 as ab

from . import kv_reference as R
from .test_gpu_cache_attention import Work

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("window", (100, 320, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31, 2 ** 40))
@pytest.mark.parametrize("sinks", (0, 4, 2 ** 31 - 1))
@pytest.mark.parametrize("lengths,queries,hq,hkv,d", [([2, 40, 0], [5, 6, 3], 4, 2, 128), ([2, 300], [80, 90], 4, 2, 128), ([1, 70], [60, 60], 2, 1, 256), ([3], [9], 2, 2, 64)])
def test_wide_windows_of_fewer_tokens_than_queries(cuda_device, lengths, queries, hq, hkv, d, sinks, window):
    """A window as wide as the page table, or as wide as numbers go, is no window, at negative positions too."""
    w = Work(cuda_device, lengths, queries, hq, hkv, d, page=32)
    got = w.run(window=window, sinks=sinks)
    w.check(got, window=window, sinks=sinks)
    if window >= w.table.shape[1] * 32:
        assert torch.equal(got, w.run())


def owners(d):
    """The token (0 to 15) that every byte of a slab of 16 tokens belongs to, from the documented order."""
    planes, j = max(1, d // 128), min(4, d // 32)
    token = torch.arange(16)
    keys = token.view(1, 16, 1).expand(planes, 16, 8 * d // planes // 16)
    half, t, odd = torch.arange(2).view(2, 1, 1, 1, 1, 1), torch.arange(4).view(1, 1, 4, 1, 1, 1), torch.arange(2).view(1, 1, 1, 1, 2, 1)
    values = (8 * half + 2 * t + odd).expand(2, 8, 4, j, 2, 2).expand(planes, 2, 8, 4, j, 2, 2)
    key_params = token.view(16, 1).expand(16, d // 16)
    value_params = (2 * torch.arange(8).view(8, 1, 1, 1, 1) + torch.arange(2).view(1, 1, 1, 2, 1)).expand(8, d // 64, 2, 2, 2)
    return torch.cat([x.reshape(-1) for x in (keys, values, key_params, value_params)])


def spoil(w, b, hidden, word):
    """Every byte of the hidden tokens (a mask over the sequence's pages) becomes that of a 16-bit word."""
    d, page = w.cache.head_dim, w.cache.page_size
    own = owners(d)
    pattern = torch.tensor([word & 255, word >> 8], dtype=torch.uint8).repeat(9 * d)
    for i in range(hidden.shape[0] // page):
        at = int(w.table[b, i])
        data = w.cache.data[at].cpu().view(w.cache.kv_heads, page // 16, 18 * d)
        gone = hidden[i * page:(i + 1) * page].view(page // 16, 16)[:, own]
        w.cache.data[at] = torch.where(gone, pattern, data).view(w.cache.kv_heads, -1).to(w.device)


@pytest.mark.parametrize("word", (0x7FFF, 0x7C00, 0xFC00))
@pytest.mark.parametrize("queries", (1, 5, 40))
@pytest.mark.parametrize("d,window,sinks", [(64, 64, 4), (128, 64, 0), (128, 50, 20), (256, 100, 17), (128, None, 0), (64, 33, 16)])
def test_what_no_query_sees_may_hold_anything(cuda_device, d, window, sinks, queries, word):
    """Keys and values, codes and scales, of tokens in front of the window, between the sinks and it, and behind the end: NaN
    and infinities there change no bit of the result."""
    w = Work(cuda_device, [1000, 905, 70], [queries] * 3, 4, 2, d, page=32, dtype=F16)
    how = dict(window=window, sinks=sinks)
    want = w.run(**how)
    w.check(want, **how)
    for b, n in enumerate(w.lengths):
        key = torch.arange(-(-n // 32) * 32)
        hidden = key >= n
        if window:
            hidden |= (key <= n - queries - window) & (key >= sinks)
        assert hidden.any()
        spoil(w, b, hidden, word)
    assert torch.equal(w.run(**how), want)


def spoil_free_memory(like):
    """Blocks of this size that the allocator hands out next hold NaN."""
    for _ in range(2):
        blocks = [torch.full_like(like, float("nan")) for _ in range(4)]
        del blocks


@pytest.mark.parametrize("starts,total,most", [([3, 5, 9, 9], 14, 4), ([0, 1, 2, 3], 3, 1), ([2, 2, 2, 2], 40, 1), ([3, 63, 110, 150], 170, 60), ([0, 6, 8, 9], 9, 2), ([0, 50, 95, 96], 96, 40),
                                               ([1, 41, 42, 130], 130, 40), ([0, 0, 1, 2], 4096, 2), ([0, 300, 500, 700], 2000, 200)])
@pytest.mark.parametrize("d,hq,hkv", [(128, 4, 2), (64, 6, 2), (256, 2, 2)])
def test_rows_of_no_sequence(cuda_device, d, hq, hkv, starts, total, most):
    """Rows in front of the first start, behind the last and beyond max_queries are zeros; the others are as without them."""
    counts = [b - a for a, b in zip(starts, starts[1:])]
    w = Work(cuda_device, [400, 120, 333], counts, hq, hkv, d, page=32)
    out, mass = R.attention(w.q, w.ks, w.vs, counts)
    want, slack = torch.zeros(2, total, hq, d, dtype=torch.float64)
    rows = []
    for a, b in zip(starts, starts[1:]):
        rows += list(range(a, min(b, a + most)))
    at = torch.tensor(rows, dtype=torch.int64)
    want[at], slack[at] = out[at - starts[0]], mass[at - starts[0]] * (2.0 ** -10 + 2e-5) + 1e-6
    q = torch.full((total, hq, d), float("nan"), dtype=BF16, device=cuda_device)
    q[starts[0]:starts[-1]] = w.q
    lengths = torch.tensor(w.lengths, dtype=torch.int32, device=cuda_device)
    spoil_free_memory(q)
    got = ab.cache_attention(q, w.cache, w.table, lengths, query_starts=torch.tensor(starts, dtype=torch.int32, device=cuda_device), max_queries=most)
    R.assert_rounded(got, want, slack)
    rest = torch.ones(total, dtype=torch.bool)
    rest[at] = False
    assert not got[rest.to(cuda_device)].any()


def test_starts_without_a_bound_and_out_of_order(cuda_device):
    """All queries is the bound where none is given; a start behind the next one is the end of an empty sequence."""
    w = Work(cuda_device, [64, 64], [2, 0], 4, 2, 64, page=16)
    lengths = torch.tensor(w.lengths, dtype=torch.int32, device=cuda_device)
    for starts in ([0, 2, 2], [0, 2, 1], [-5, 2, 2 ** 31 - 1]):
        spoil_free_memory(w.q)
        w.check(ab.cache_attention(w.q, w.cache, w.table, lengths, query_starts=torch.tensor(starts, dtype=torch.int32, device=cuda_device)))
    w = Work(cuda_device, [300, 70], [90, 40], 4, 2, 64, page=16)
    lengths = torch.tensor(w.lengths, dtype=torch.int32, device=cuda_device)
    w.check(ab.cache_attention(w.q, w.cache, w.table, lengths, query_starts=w.starts))


def test_queries_without_sequences(cuda_device):
    cache = ab.QuantizedKVCache(2, 2, 64, page_size=16, device=cuda_device)
    q = torch.ones(5, 4, 64, dtype=F16, device=cuda_device)
    none = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    spoil_free_memory(q)
    got = ab.cache_attention(q, cache, none.view(0, 3), none, query_starts=torch.zeros(1, dtype=torch.int32, device=cuda_device))
    assert got.shape == q.shape and not got.any()
