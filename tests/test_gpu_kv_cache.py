"""The 4-bit cache, norms and rotations against their definitions in 64 bits."""
import pytest
import torch

import atlasinfer_b200 as ab
from atlasinfer_b200 import _capi

from . import kv_reference as R

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(shape, dtype, seed, device):
    return torch.randn(shape, generator=gen(seed)).to(dtype).to(device)


def slots_of(count, total, seed, device, dtype=torch.int64):
    return torch.randperm(total, generator=gen(seed))[:count].to(dtype).to(device)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("tokens,heads,d,page", [(1, 1, 64, 16), (7, 3, 128, 48), (130, 2, 256, 64), (33, 5, 64, 32), (1000, 4, 128, 16), (3, 1, 256, 128)])
def test_store_and_load(cuda_device, tokens, heads, d, page, dtype):
    pages = tokens // page + 3
    cache = ab.QuantizedKVCache(pages, heads, d, page_size=page, device=cuda_device)
    k, v = (randn((tokens, heads, d), dtype, s, cuda_device) * (1 + 3 * s) for s in (0, 1))
    slots = slots_of(tokens, pages * page, 2, cuda_device, torch.int64 if tokens % 2 else torch.int32)
    cache.store(k, v, slots)
    kc, vc = cache.load(slots)
    # 16-bit numbers divide into steps of 7 bits exactly, ties included: every stored number is determined
    assert torch.equal(kc.cpu().double(), R.stored(k)) and torch.equal(vc.cpu().double(), R.stored(v))
    kb, vb = cache.load(slots, dtype=BF16)
    assert torch.equal(kb, kc.to(BF16)) and torch.equal(vb, vc.to(BF16))
    again = ab.QuantizedKVCache(pages, heads, d, page_size=page, device=cuda_device)
    again.store(kc, vc, slots)
    kk, vv = again.load(slots)
    assert float((kk.double() - kc.double()).abs().max()) <= float(R.steps(kc).max()) / 2


@pytest.mark.parametrize("d", (64, 128, 256))
def test_bytes(cuda_device, d):
    """The documented place of every number."""
    page, heads = 32, 2
    cache = ab.QuantizedKVCache(2, heads, d, page_size=page, device=cuda_device)
    k, v = (randn((64, heads, d), F16, s, cuda_device) for s in (3, 4))
    cache.store(k, v, torch.arange(64, device=cuda_device))
    data = cache.data.cpu().view(2, heads, page // 16, 18 * d)
    (ck, sk, zk), (cv, sv, zv) = R.groups(k), R.groups(v)
    ck, cv = ck.flatten(-2).int(), cv.flatten(-2).int()
    wide, words = min(d, 128), min(d, 128) // 32
    half = lambda b: b.contiguous().view(F16).item()  # noqa: E731
    for token, head, ch in [(0, 0, 0), (1, 1, 1), (15, 0, d - 1), (16, 1, 63), (37, 0, d // 2 + 5), (63, 1, d - 64 + 17), (22, 0, 31)]:
        slab, tok, plane, c = data[token // page, head, token % page // 16], token % 16, ch // wide, ch % wide
        n = (((tok * 4 + c % 32 // 8) * words + c // 32) * 2 + c % 2) * 4 + c % 8 // 2 + plane * 16 * wide
        assert int(slab[n // 2]) >> (4 * (n % 2)) & 15 == int(ck[token, head, ch])
        n = ((((tok // 8 * 8 + c % 32 // 4) * 4 + tok % 8 // 2) * words + c // 32) * 2 + tok % 2) * 4 + c % 4 + plane * 16 * wide
        assert int(slab[8 * d + n // 2]) >> (4 * (n % 2)) & 15 == int(cv[token, head, ch])
        at = 16 * d + (tok * (d // 64) + ch // 64) * 4
        assert half(slab[at:at + 2]) == float(sk[token, head, ch // 64, 0]) and half(slab[at + 2:at + 4]) == 1024 + float(zk[token, head, ch // 64, 0])
        at = 17 * d + (tok // 2 * (d // 64) + ch // 64) * 8 + tok % 2 * 2
        assert half(slab[at:at + 2]) == float(sv[token, head, ch // 64, 0]) and half(slab[at + 4:at + 6]) == 1024 + float(zv[token, head, ch // 64, 0])


def test_special_numbers(cuda_device):
    """Groups of zeros, of one number, without a sign, tiny, huge, with infinities and NaN: finite, and as defined."""
    inf, nan = float("inf"), float("nan")
    rows = [torch.zeros(64), torch.full((64,), 3.0), torch.full((64,), -0.7), torch.linspace(5, 6, 64), torch.linspace(-6, -5, 64), torch.full((64,), 6e-8),
            torch.linspace(-60000, 60000, 64), torch.linspace(0, 65504, 64), torch.tensor([inf] + 63 * [1.0]), torch.tensor([-inf, inf] + 62 * [2.0]),
            torch.tensor([nan] + 63 * [1.5]), torch.full((64,), nan)]
    for dtype, more in ((F16, []), (BF16, [torch.full((64,), 3e38), torch.linspace(-1e30, 1e-30, 64)])):
        x = torch.stack(rows + more).to(dtype).to(cuda_device)[:, None]
        cache = ab.QuantizedKVCache(1, 1, 64, page_size=16, device=cuda_device)
        slots = torch.arange(x.shape[0], device=cuda_device)
        cache.store(x, x.flip(0), slots)
        k, v = cache.load(slots)
        assert torch.equal(k.cpu().double(), R.stored(x)) and torch.equal(v.cpu().double(), R.stored(x.flip(0)))
        assert bool(k.isfinite().all())


def test_slots_outside(cuda_device):
    cache = ab.QuantizedKVCache(3, 2, 128, page_size=16, device=cuda_device)
    k, v = (randn((6, 2, 128), BF16, s, cuda_device) for s in (0, 1))
    slots = torch.tensor([-1, 5, 48, 47, 1 << 40, -(1 << 40)], device=cuda_device)
    cache.store(k, v, slots)
    kc, vc = cache.load(slots)
    for i, there in enumerate((False, True, False, True, False, False)):
        assert torch.equal(kc[i].cpu().double(), R.stored(k[i]) if there else torch.zeros(2, 128, dtype=torch.float64))
        assert torch.equal(vc[i].cpu().double(), R.stored(v[i]) if there else torch.zeros(2, 128, dtype=torch.float64))
    rest = torch.tensor([s for s in range(48) if s not in (5, 47)], device=cuda_device)
    assert not cache.load(rest)[0].any() and not cache.load(rest)[1].any()   # nothing else was touched
    cache.store(k[:0], v[:0], slots[:0])
    assert cache.load(slots[:0])[0].shape == (0, 2, 128)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("tokens,hq,hkv,d,rotary,interleaved,norm,offset", [
    (1, 1, 1, 64, 64, False, None, 0.0), (5, 6, 2, 64, 32, True, "same", 0.0), (3, 9, 3, 128, 48, False, "fp32", 1.0), (17, 5, 5, 128, 128, False, "k", 0.0),
    (129, 8, 1, 256, 256, True, "same", 1.0), (2, 7, 7, 256, 16, False, "q", 0.0), (1, 64, 8, 128, 0, False, "same", 0.0), (600, 16, 2, 128, 128, False, "same", 0.0)])
def test_norm_rotate(cuda_device, tokens, hq, hkv, d, rotary, interleaved, norm, offset, dtype):
    x = randn((tokens, (hq + 2 * hkv) * d), dtype, 5, cuda_device) * 3
    q, k, v = (y.unflatten(-1, (-1, d)) for y in x.split([hq * d, hkv * d, hkv * d], -1))
    table = ab.rotary_table(1000, rotary, device=cuda_device) if rotary else None
    positions = torch.randint(0, 1000, (tokens,), generator=gen(6)).to(torch.int32 if tokens % 2 else torch.int64).to(cuda_device) if rotary else None
    wtype = torch.float32 if norm == "fp32" else dtype
    qw = None if norm in (None, "k") else randn((d,), wtype, 7, cuda_device)
    kw = None if norm in (None, "q") else randn((d,), wtype, 8, cuda_device)
    how = dict(table=table, positions=positions, eps=1e-5, weight_offset=offset, interleaved=interleaved)
    got_q, got_k = ab.norm_rotate(q, k, q_weight=qw, k_weight=kw, **how)
    # in 32 bits: the sum of D squares to D / 2 units in the last place (in practice far fewer), then five roundings
    for got, src, w in ((got_q, q, qw), (got_k, k, kw)):
        want = R.turned(src, w, **how)
        assert got.is_contiguous() and got.shape == src.shape
        R.assert_rounded(got, want, want.abs().amax(-1, keepdim=True) * (d / 2 + 5) * 2.0 ** -24)
    # the same, into a cache: the queries are the same bits, keys at most half a step (and that error) from the definition
    cache = ab.QuantizedKVCache(tokens // 16 + 1, hkv, d, page_size=16, device=cuda_device)
    slots = slots_of(tokens, cache.num_slots, 9, cuda_device)
    stored_q = ab.norm_rotate_store(q, k, v, cache, slots, q_weight=qw, k_weight=kw, **how)
    assert torch.equal(stored_q, got_q)
    kc, vc = cache.load(slots)
    assert torch.equal(vc.cpu().double(), R.stored(v))
    want = R.turned(k, kw, **how)
    err = (kc.cpu().double() - want).abs()
    # (the range of a group has a step of 15.117 of its 15 ninths at most: rounded up to 7 bits)
    assert bool((err <= R.steps(want) * (0.5 * (1 + 2.0 ** -6) + 1e-3) + want.abs() * 1e-5).all())
    same = (kc.cpu().double() == R.stored(want.float())).double().mean()
    assert float(same) > 0.999, float(same)   # one in 10^6 lies within 2^-20 of a tie; a scale one in 10^4


def test_positions_outside_the_table(cuda_device):
    q, k = randn((4, 2, 64), F16, 0, cuda_device), randn((4, 1, 64), F16, 1, cuda_device)
    table = ab.rotary_table(8, 32, device=cuda_device)
    got_q, got_k = ab.norm_rotate(q, k, table, torch.tensor([7, 8, -1, 0], device=cuda_device))
    assert bool(got_q[[1, 2], :, :32].isnan().all()) and bool(got_k[[1, 2], :, :32].isnan().all())
    assert bool(got_q[[0, 3]].isfinite().all()) and torch.equal(got_q[..., 32:], q[..., 32:])


def test_strides_and_addresses(cuda_device):
    """Heads first, odd addresses, every other token: read in place or copied, the results are those of the dense tensors."""
    table, positions = ab.rotary_table(64, 64, device=cuda_device), torch.arange(6, device=cuda_device)
    base_q, base_k = randn((4, 12, 64), BF16, 0, cuda_device), randn((2, 12, 64), BF16, 1, cuda_device)
    q, k = base_q.transpose(0, 1)[::2], base_k.transpose(0, 1)[::2]
    want = ab.norm_rotate(q.contiguous(), k.contiguous(), table, positions)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device=cuda_device)[1:].view(q.shape)
    odd.copy_(q)
    wide = torch.empty(6, 4, 128, dtype=BF16, device=cuda_device)[..., ::2]
    wide.copy_(q)
    for qq in (q, odd, wide, q.contiguous()):
        got = ab.norm_rotate(qq, k, table, positions)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = ab.norm_rotate(q[:1].expand(6, 4, 64), k, table, positions)   # a broadcast token
    assert torch.equal(one[0][0], want[0][0])


def test_far_pages(cuda_device):
    """Offsets beyond 32 bits: the last pages of a cache of 5 GB."""
    heads, d, page = 8, 256, 64
    pages = (5 << 30) // (heads * ab.QuantizedKVCache.page_bytes(d, page))
    data = torch.empty(pages, heads, ab.QuantizedKVCache.page_bytes(d, page), dtype=torch.uint8, device=cuda_device)
    cache = ab.QuantizedKVCache(pages, heads, d, page_size=page, data=data)
    k, v = (randn((40, heads, d), F16, s, cuda_device) for s in (0, 1))
    slots = torch.arange(cache.num_slots - 40, cache.num_slots, device=cuda_device)
    cache.store(k, v, slots)
    kc, vc = cache.load(slots)
    assert torch.equal(kc.cpu().double(), R.stored(k)) and torch.equal(vc.cpu().double(), R.stored(v))
    q = randn((1, 16, d), F16, 2, cuda_device)
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=cuda_device)
    # (the last page holds those 40 tokens at its end: its first 24 are another sequence's)
    cache.store(k[:24], v[:24], slots[:24] - 24)
    got = ab.cache_attention(q, cache, table, torch.tensor([64], dtype=torch.int32, device=cuda_device))
    ks, vs = (torch.cat([R.stored(x[:24]), R.stored(x)]) for x in (k, v))
    out, mass = R.attention(q, [ks], [vs], [1])
    R.assert_rounded(got, out, mass * (2.0 ** -10 + 2e-5))


def test_c_entries_refuse(cuda_device):
    L = _capi.load()
    a = _capi.Tokens(dtype=0, q_heads=1, kv_heads=1, head_dim=64, tokens=1)
    assert L.atlas_norm_rotate(a, None) == _capi.ERR_BAD_ARGUMENT and b"null" in L.atlas_last_error()
    x = torch.zeros(64, dtype=F16, device=cuda_device)
    a.q = a.k = a.q_out = a.k_out = x.data_ptr()
    a.q = x.data_ptr() + 2
    assert L.atlas_norm_rotate(a, None) == _capi.ERR_BAD_ARGUMENT and b"16 bytes" in L.atlas_last_error()
