"""Members of a fused group give what the module alone gives, whatever happens between their calls."""
import pytest
import torch

import atlasinfer_b200 as ab

from . import decoder_reference as D
from .kv_reference import assert_rounded
from .test_gpu_fused_linear import module, randn

pytestmark = pytest.mark.gpu

F16 = torch.float16


def group(device, count=3):
    """``(modules, weights)`` of a group."""
    mods, weights = zip(*(module(96 + 64 * i, 256, 20 + i, device) for i in range(count)))
    ab.fuse_linears(mods)
    return mods, weights


def check(mod, w, x, y=None, bias=None):
    b = mod.bias if bias is None else bias
    assert_rounded(mod(x) if y is None else y, *D.product(x, w, None if b is None else b.half()))   # (the kernels add an fp16 bias)


@pytest.mark.parametrize("m", (1, 40))
def test_inference_mode(cuda_device, m):
    """Inputs that do not count how often they are written to, between the members' calls too."""
    mods, weights = group(cuda_device)
    with torch.inference_mode():
        x = randn((m, 256), F16, 0, cuda_device)
        for mod, w in zip(mods, weights):
            check(mod, w, x)
        first = mods[0](x)
        before = x.clone()
        x.copy_(randn((m, 256), F16, 1, cuda_device))
        check(mods[0], weights[0], before, first)
        for mod, w in zip(mods[1:], weights[1:]):
            check(mod, w, x)
    x = randn((m, 256), F16, 2, cuda_device)   # outside it the members share a launch again
    launches = mods[0]._group.launches
    for mod, w in zip(mods, weights):
        check(mod, w, x)
    assert mods[0]._group.launches == launches + 1
