"""Attention over the 4-bit cache against its definition in 64 bits."""
import pytest
import torch

import atlasinfer_b200 as ab

from . import kv_reference as R

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


class Work:
    """Sequences in shuffled pages, and queries at their ends."""

    def __init__(self, device, lengths, queries, hq, hkv, d, page=16, dtype=BF16, seed=0, lean=0.0, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.queries, self.device = lengths, queries, device
        need = [-(-n // page) for n in lengths]
        self.cache = ab.QuantizedKVCache(sum(need) + spare, hkv, d, page_size=page, device=device)
        order = torch.randperm(sum(need) + spare, generator=g)
        self.table = torch.full((len(lengths), max(need + [1])), -1, dtype=torch.int32)
        self.ks, self.vs = [], []
        at = 0
        direction = torch.randn(hkv, d, generator=g)
        for b, n in enumerate(lengths):
            pages = order[at:at + need[b]]
            at += need[b]
            self.table[b, :need[b]] = pages.int()
            k, v = (torch.randn(n, hkv, d, generator=g) for _ in range(2))
            if n:
                k[0] += lean * direction
            k, v = k.to(dtype), v.to(dtype)
            if n:
                slots = (pages[torch.arange(n) // page] * page + torch.arange(n) % page).to(device)
                self.cache.store(k.to(device), v.to(device), slots)
            self.ks.append(R.stored(k))
            self.vs.append(R.stored(v))
        self.q = torch.randn(sum(queries), hkv, hq // hkv, d, generator=g) + lean * direction[:, None]
        self.q = self.q.flatten(1, 2).to(dtype).to(device)
        self.table = self.table.to(device)
        self.starts = torch.tensor([sum(queries[:i]) for i in range(len(queries) + 1)], dtype=torch.int32, device=device)

    def run(self, q=None, **how):
        lengths = torch.tensor(self.lengths, dtype=torch.int32, device=self.device)
        if len(set(self.queries)) > 1:
            how = dict(query_starts=self.starts, max_queries=max(self.queries), **how)
        return ab.cache_attention(self.q if q is None else q, self.cache, self.table, lengths, **how)

    def check(self, got=None, **how):
        got = self.run(**how) if got is None else got
        assert got.shape == self.q.shape and got.dtype == self.q.dtype
        out, mass = R.attention(self.q, self.ks, self.vs, self.queries, **how)
        # weights are fp16 over the sum of what they were rounded to: 2^-10 relative; scores are sums in 32 bits
        R.assert_rounded(got, out, mass * (2.0 ** -10 + 2e-5) + 2.0 ** -30 * max(self.lengths))


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 4), (64, 9, 3), (128, 8, 1), (128, 14, 2), (128, 32, 2), (256, 2, 2), (256, 32, 4), (128, 3, 1), (256, 24, 1)])
def test_one_token(cuda_device, d, hq, hkv, dtype):
    lengths = [1, 2, 15, 16, 17, 33, 200, 47, 0, 64]
    Work(cuda_device, lengths, [1] * len(lengths), hq, hkv, d, dtype=dtype, page=32).check()


@pytest.mark.parametrize("page", (16, 48, 64, 128))
@pytest.mark.parametrize("lengths", [[1], [5000], [3001, 1, 4097, 0, 777], [100] * 37, [1, 1, 1, 9000]])
def test_lengths_and_pages(cuda_device, lengths, page):
    Work(cuda_device, lengths, [1] * len(lengths), 8, 2, 128, page=page, lean=0.5).check()


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("lengths,queries,hq,hkv,d", [
    ([40, 7, 300], [2, 2, 2], 8, 8, 64), ([40, 7, 300, 16], [5, 1, 3, 16], 8, 2, 128), ([33], [33], 4, 4, 128), ([257], [129], 6, 2, 64),
    ([100, 500], [100, 130], 8, 1, 256), ([700, 3, 64, 0, 20], [300, 3, 1, 0, 20], 8, 2, 128), ([2, 5], [4, 9], 2, 1, 128), ([130], [130], 1, 1, 64),
    ([1025], [1025], 2, 2, 128), ([600, 600], [200, 200], 5, 1, 256), ([90, 0, 40], [0, 0, 40], 4, 2, 64)])
def test_many_queries(cuda_device, lengths, queries, hq, hkv, d, dtype):
    """Causal rows; more queries than tokens leaves the first rows without any."""
    Work(cuda_device, lengths, queries, hq, hkv, d, dtype=dtype, page=48).check()


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("lengths,queries,hq,hkv,d,window", [([3000, 2100], [20, 33], 8, 2, 128, None), ([5000], [60], 2, 1, 64, None), ([2500, 70, 0], [30, 40, 9], 16, 2, 256, None),
                                                             ([4000, 3100], [100, 90], 4, 2, 128, 700)])
def test_split_contexts(cuda_device, lengths, queries, hq, hkv, d, window, dtype):
    """Some tens of rows over long contexts: the tokens are split among CTAs and joined."""
    Work(cuda_device, lengths, queries, hq, hkv, d, dtype=dtype, page=64, lean=0.3).check(window=window, sinks=5 if window else 0)


@pytest.mark.parametrize("rows", (8, 9, 16, 17, 25, 32, 33))
@pytest.mark.parametrize("d", (64, 128, 256))
def test_rows_of_a_group(cuda_device, rows, d):
    """Every number of row tiles, few tokens and many (with room in the page table, which the choice of the kernel goes by)."""
    w = Work(cuda_device, [2000, 33, 500], [1, 1, 1], rows, 1, d, page=16)
    w.check()
    w.table = torch.cat([w.table, torch.full((3, 5000), -1, dtype=torch.int32, device=cuda_device)], 1)
    w.check()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 4), (100, 16), (100, 33), (5000, 7), (64, 500), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("lengths,queries,hq,hkv,d", [([1, 18, 500, 77, 1200], [1] * 5, 8, 2, 128), ([300, 40, 801], [90, 3, 260], 4, 1, 64), ([400], [400], 2, 2, 256)])
def test_window_and_sinks(cuda_device, lengths, queries, hq, hkv, d, window, sinks):
    Work(cuda_device, lengths, queries, hq, hkv, d, page=32).check(window=window, sinks=sinks)


@pytest.mark.parametrize("queries", (1, 40))
def test_pages_without_visible_tokens_are_not_read(cuda_device, queries):
    """Freed pages may have any entry, and everything that no query sees may hold anything (here NaN and infinite scales)."""
    w = Work(cuda_device, [1000, 900], [queries, queries], 4, 2, 128, page=16)
    want = w.run(window=64, sinks=4)
    w.check(want, window=64, sinks=4)
    lens = torch.tensor(w.lengths)
    for b, n in enumerate(w.lengths):
        first = (n - queries - 64 + 1) // 16
        used = w.table[b, :-(-n // 16)].long()
        w.cache.data[used[1:first]] = 0xFF
        w.table[b, 1:first] = torch.tensor([-1, 2 ** 31 - 1, w.cache.num_pages, -(2 ** 31)] * 20, dtype=torch.int32, device=cuda_device)[:first - 1]
        spoil_after(w.cache, int(used[-1]), n - (n - 1) // 16 * 16)
    spare = torch.ones(w.cache.num_pages, dtype=torch.bool)
    for b, n in enumerate(w.lengths):
        spare[w.table[b, (w.table[b] >= 0) & (w.table[b] < w.cache.num_pages)].long().cpu()] = False
    w.cache.data[spare.to(cuda_device)] = 0xFF
    assert torch.equal(w.run(window=64, sinks=4), want)
    assert int(lens.max()) == 1000


def spoil_after(cache, page, count):
    """Sets every byte of a 16-token page of heads of 128 that belongs to its tokens from ``count`` on."""
    data = cache.data[page]
    gone = torch.arange(16, device=data.device) >= count
    data[:, :1024].view(-1, 16, 64)[:, gone] = 0xFF
    data[:, 16 * 128:17 * 128].view(-1, 16, 8)[:, gone] = 0xFF
    values = data[:, 1024:2048].view(-1, 2, 8, 4, 4, 2, 2)     # half, g, t, j, odd, byte
    params = data[:, 17 * 128:].view(-1, 8, 2, 2, 2, 2)        # pair, group, scale or zero, odd, byte
    for token in range(count, 16):
        values[:, token // 8, :, token % 8 // 2, :, token % 2] = 0xFF
        params[:, token // 2, :, :, token % 2] = 0xFF


@pytest.mark.parametrize("word", (0x7FFF, 0x7E00, 0xFC00, 0xFFFF))
@pytest.mark.parametrize("queries", (1, 40))
def test_hidden_tokens_of_a_slab_may_hold_anything(cuda_device, queries, word):
    """What the window has left behind within the first slab that it still sees: no pattern there hides the slab."""
    w = Work(cuda_device, [1000, 905], [queries, queries], 4, 2, 128, page=16)
    want = w.run(window=64)
    w.check(want, window=64)
    for b, n in enumerate(w.lengths):
        first = n - queries - 63   # (the first query's first key)
        assert first % 16
        data = w.cache.data[int(w.table[b, first // 16])]          # [head, bytes]: keys of tokens in front of it
        patch = data.view(torch.int16)
        patch[:, 16 * 64:17 * 64].view(-1, 16, 4)[:, :first % 16] = word - (1 << 16 if word > 0x7FFF else 0)
        w.cache.data[int(w.table[b, first // 16])] = data
    assert torch.equal(w.run(window=64), want)


@pytest.mark.parametrize("queries", (1, 50))
def test_unknown_pages_count_as_hidden(cuda_device, queries):
    w = Work(cuda_device, [200, 64], [queries] * 2, 4, 2, 64, page=16)
    w.table[0, 2], w.table[0, 5], w.table[1, :] = -1, w.cache.num_pages, -7
    got = w.run()
    keep = torch.ones(200, dtype=torch.bool)
    keep[32:48] = keep[80:96] = False
    hidden = torch.where(keep, 0.0, -1.0)[:, None, None]
    # the tokens of unknown pages removed, the others at their positions: by weights of zero in the definition
    q = w.q[:queries].cpu().double()
    k, v = w.ks[0], w.vs[0]
    s = torch.einsum("nhrd,khd->nhrk", q.unflatten(1, (2, 2)), k) / 8
    seen = (torch.arange(200) <= 200 - queries + torch.arange(queries)[:, None]) & keep
    p = torch.softmax(s.masked_fill(~seen[:, None, None], -float("inf")), -1)
    out, mass = (torch.einsum("nhrk,khd->nhrd", p, x).flatten(1, 2) for x in (v, v.abs()))
    R.assert_rounded(got[:queries], out, mass * (2.0 ** -10 + 2e-5) + 1e-6)
    assert not got[queries:].any() and hidden.shape[0] == 200


def test_scores_of_any_size(cuda_device):
    """Far apart (one key takes all), all equal, and queries of 1e-30 and 1e30."""
    for size in (0.0, 1e-30, 60.0, 1e30):
        w = Work(cuda_device, [70, 300], [1, 1], 8, 2, 128, dtype=BF16, lean=1.0)
        w.q = (w.q.float() * size).to(BF16)
        w.check(scale=0.1 if size < 1e9 else 1e-31)


def test_infinite_and_nan_queries(cuda_device):
    """A query with NaN makes its own row NaN and no other."""
    for queries in (1, 30):
        w = Work(cuda_device, [90, 90], [queries] * 2, 4, 2, 128, dtype=F16)
        want = w.run()
        w.q[queries, 1, 5] = float("nan")
        got = w.run()
        assert bool(got[queries, 1].isnan().all())
        got[queries, 1] = want[queries, 1]
        assert torch.equal(got, want)


def test_strided_queries_and_same_bits(cuda_device):
    w = Work(cuda_device, [500, 2000, 30], [1, 1, 1], 8, 2, 128)
    fused = torch.randn(3, 24 * 128, device=cuda_device).to(BF16)
    view = fused[:, 256:256 + 1024].unflatten(-1, (8, 128))
    want = w.run(view.contiguous())
    for _ in range(3):
        assert torch.equal(w.run(view), want)
    heads_first = view.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(w.run(heads_first), want)
    odd = torch.empty(view.numel() + 1, dtype=BF16, device=cuda_device)[1:].view(view.shape).copy_(view)
    assert torch.equal(w.run(odd), want)


@pytest.mark.parametrize("queries", (1, 3, 70))
def test_graph_replayed_for_other_lengths(cuda_device, queries):
    """The lengths are read on the device: a captured call serves any."""
    w = Work(cuda_device, [400, 300, 200], [queries] * 3, 8, 2, 64)
    lengths = torch.tensor([80, 300, 90], dtype=torch.int32, device=cuda_device)
    call = lambda: ab.cache_attention(w.q, w.cache, w.table, lengths)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for new in ([80, 300, 90], [400, 0, 200], [1, 1, 1]):
        lengths.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        ref, mass = R.attention(w.q, [k[:n] for k, n in zip(w.ks, new)], [v[:n] for v, n in zip(w.vs, new)], w.queries)
        R.assert_rounded(out, ref, mass * (2.0 ** -10 + 2e-5) + 1e-6)


def test_other_streams(cuda_device):
    """Two streams attend to one cache at a time; every call has a workspace of its own."""
    w = Work(cuda_device, [3000, 2500], [1, 1], 8, 2, 128)
    want = w.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for s, g in zip(streams, got):
            with torch.cuda.stream(s):
                g.append(w.run())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for g in got for x in g)


def test_lengths_that_do_not_fit(cuda_device):
    """Lengths beyond the page table end with it, negative ones are none; starts out of order give empty sequences."""
    w = Work(cuda_device, [64, 64], [1, 1], 4, 2, 64, page=16)
    call = lambda n, **how: ab.cache_attention(w.q, w.cache, w.table, torch.tensor(n, dtype=torch.int32, device=cuda_device), **how)  # noqa: E731
    full = call([64, 64])
    assert torch.equal(call([10 ** 9, 64]), full)
    none = call([-5, 64])
    assert not none[0].any() and torch.equal(none[1], full[1])
    starts = torch.tensor([0, 2, 1], dtype=torch.int32, device=cuda_device)
    odd = call([64, 64], query_starts=starts, max_queries=2)
    assert odd.shape == full.shape


def test_decode_step(cuda_device):
    """A layer's step as a model runs it: fused q/k/v linear, norm and rotation into the cache, attention, output linear."""
    hq, hkv, d, hidden, batch = 8, 2, 64, 512, 3
    g = torch.Generator().manual_seed(0)
    mods = [ab.QuantizedLinear(ab.quantize_tensor((torch.randn(n, hidden, generator=g) * 0.05).half().to(cuda_device)), None) for n in (hq * d, hkv * d, hkv * d, hidden)]
    ab.fuse_linears(mods[:3])
    cache = ab.QuantizedKVCache(8, hkv, d, page_size=16, device=cuda_device)
    pages = torch.tensor([[3, 5], [0, 7], [6, 1]], dtype=torch.int32, device=cuda_device)
    table = ab.rotary_table(64, d, device=cuda_device)
    ks, vs = [[] for _ in range(batch)], [[] for _ in range(batch)]
    for step in range(20):
        x = torch.randn(batch, hidden, generator=g).to(BF16).to(cuda_device)
        q, k, v = (mod(x).unflatten(-1, (-1, d)) for mod in mods[:3])
        at = torch.full((batch,), step, device=cuda_device)
        slots = pages[:, step // 16].long() * 16 + step % 16
        turned = ab.norm_rotate_store(q, k, v, cache, slots, table, at)
        lengths = (at + 1).int()
        out = ab.cache_attention(turned, cache, pages, lengths)
        y = mods[3](out.flatten(1))
        assert y.shape == (batch, hidden) and bool(y.isfinite().all())
        kc, vc = cache.load(slots)
        for b in range(batch):
            ks[b].append(kc[b].cpu().double())
            vs[b].append(vc[b].cpu().double())
        ref, mass = R.attention(turned, [torch.stack(x) for x in ks], [torch.stack(x) for x in vs], [1] * batch)
        R.assert_rounded(out, ref, mass * (2.0 ** -10 + 2e-5) + 1e-6)
