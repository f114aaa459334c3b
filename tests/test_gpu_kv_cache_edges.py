"""The 4-bit cache at the edges of positions and of numbers."""
import pytest
import torch

import atlasinfer_b200 as ab

from . import kv_reference as R

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("d,rotary,interleaved,norm", [(64, 32, False, False), (128, 128, True, False), (256, 64, False, True), (128, 48, True, True)])
def test_stored_keys_of_unknown_positions(cuda_device, d, rotary, interleaved, norm):
    """The rotated channels of such a token are NaN in its query and stored as zeros in its key; the others, and its value,
    are as ever, and so are the tokens beside it."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(5, h, d, generator=g).to(BF16).to(cuda_device) for h in (4, 2, 2))
    weight = (1 + 0.1 * torch.randn(d, generator=g)).to(BF16).to(cuda_device) if norm else None
    table = ab.rotary_table(8, rotary, device=cuda_device)
    positions = torch.tensor([7, 8, -1, 0, 2 ** 40], device=cuda_device)
    lost, kept = [1, 2, 4], [0, 3]
    cache = ab.QuantizedKVCache(1, 2, d, page_size=16, device=cuda_device)
    slots = torch.arange(5, device=cuda_device)
    out = ab.norm_rotate_store(q, k, v, cache, slots, table, positions, q_weight=weight, k_weight=weight, interleaved=interleaved)
    how = dict(table=table, positions=positions.clamp(0, 7), interleaved=interleaved)
    want_q, want_k = R.turned(q, weight, **how), R.turned(k, weight, **how)
    want_k[lost, :, :rotary] = float("nan")
    assert bool(out[lost, :, :rotary].isnan().all())
    slack = want_q.abs().amax(-1, keepdim=True) * (d / 2 + 5) * 2.0 ** -24
    R.assert_rounded(out[kept], want_q[kept], slack[kept])
    R.assert_rounded(out[lost][..., rotary:], want_q[lost][..., rotary:], slack[lost])
    kc, vc = cache.load(slots)
    assert torch.equal(vc.cpu().double(), R.stored(v))
    assert not kc[lost, :, :rotary].any() and bool(kc.isfinite().all())
    steps = R.steps(want_k)
    want_k = torch.where(want_k.isnan(), torch.zeros_like(want_k), want_k)
    # half a step of a fifteenth of the range, rounded up to 7 bits, and the error of what is stored
    assert bool(((kc.cpu().double() - want_k).abs() <= steps * (0.5 * (1 + 2.0 ** -6) + 1e-3) + want_k.abs() * 1e-5).all())


def wide_groups(dtype):
    """Groups of every width up to twice 65280, and the ends of what is stored whole."""
    g = torch.Generator().manual_seed(1)
    rows = []
    for lo, hi in [(0, 65280), (-65280, 0), (-32640, 32640), (-4352, 60928), (-60928, 4352), (-1, 65216), (-60000, 60000), (-65280, 65280), (-40000, 30000), (-2000, 65000),
                   (-65000, 2000), (-3e-6, 1e-6), (-1e-3, 3e-3)]:
        x = lo + (hi - lo) * torch.rand(64, generator=g)
        x[0], x[1] = lo, hi
        rows.append(x)
    rows += [torch.tensor([float("inf"), -1.0] + 62 * [300.0]), torch.tensor([float("-inf"), float("inf")] + 62 * [-9000.0])]
    return torch.stack(rows).to(dtype)[:, None]


@pytest.mark.parametrize("dtype", (F16, BF16))
def test_ranges_that_are_stored_whole(cuda_device, dtype):
    """Half a step at most for ranges up to 65280; beyond, the low end is kept and the rest is the largest that the group holds."""
    x = wide_groups(dtype)
    cache = ab.QuantizedKVCache(2, 1, 64, page_size=16, device=cuda_device)
    slots = torch.arange(x.shape[0], device=cuda_device)
    cache.store(x.to(cuda_device), x.flip(0).to(cuda_device), slots)
    k, v = (y.cpu().double()[:, 0] for y in cache.load(slots))
    assert torch.equal(v.flip(0), k)
    x = x.double()[:, 0].clamp(-65280, 65280)
    lo, hi = x.amin(1).clamp(max=0), x.amax(1).clamp(min=0)
    whole = 0
    for i in range(x.shape[0]):
        step = float(hi[i] - lo[i]) / 15
        if hi[i] - lo[i] <= 65280:
            # (a step rounded up to 7 bits is less than 2^-6 longer, and never less than 2^-18)
            assert bool(((x[i] - k[i]).abs() <= max(step * (1 + 2.0 ** -6), 2.0 ** -18) / 2).all())
            whole += 1
        else:
            top = 4352.0 * (15 - min(15, round(-float(lo[i]) / 4352)))
            above = x[i] > top
            assert bool((k[i][above] == top).all()) and bool(((x[i] - k[i])[~above].abs() <= 2176).all())
    assert 7 <= whole < x.shape[0] - 3
