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
