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
