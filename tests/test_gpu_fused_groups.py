"""Members of a fused group give what the module alone gives, whatever happens between their calls."""
import copy
import threading

import pytest
import torch

import atlasinfer_b200 as ab

from . import decoder_reference as D
from .kv_reference import assert_rounded
from .test_gpu_fused_linear import module, randn
from .test_gpu_plain_launch import _edges

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


@pytest.mark.parametrize("m", (1, 40))
def test_members_on_streams_of_their_own(cuda_device, m):
    """A member that is called on another stream than the one before it launches the product there."""
    mods, weights = group(cuda_device)
    x = randn((m, 256), F16, 0, cuda_device)
    for mod in mods:
        mod(x)
    torch.cuda.synchronize(cuda_device)
    launches = mods[0]._group.launches
    streams, outs = [torch.cuda.Stream(cuda_device) for _ in mods], []
    for mod, s in zip(mods, streams):
        with torch.cuda.stream(s):
            outs.append(mod(x))
    assert mods[0]._group.launches == launches + len(mods)
    torch.cuda.synchronize(cuda_device)
    for mod, w, y in zip(mods, weights, outs):
        check(mod, w, x, y)


def test_outputs_may_be_written_to(cuda_device):
    """In place, with gradients of what is added."""
    mods, weights = group(cuda_device)
    x = randn((3, 256), F16, 0, cuda_device)
    outs = [mod(x) for mod in mods]
    more = torch.ones(3, 160, dtype=F16, device=cuda_device, requires_grad=True)
    outs[1] += 2 * more
    outs[1].sum().backward()
    assert bool((more.grad == 2).all())
    check(mods[0], weights[0], x, outs[0])
    check(mods[2], weights[2], x, outs[2])


@pytest.mark.parametrize("m", (1, 40))
def test_members_inside_and_outside_a_graph(cuda_device, m):
    """A captured member is computed by the graph, and one outside it is not taken from the graph's memory."""
    mods, weights = group(cuda_device)
    x = randn((m, 256), F16, 0, cuda_device)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        for mod in mods:
            mod(x)
        mods[0](x)   # (only this one: the product of all of them is at hand)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = mods[1](x)
        outside = mods[2](x)
    torch.cuda.synchronize(cuda_device)
    check(mods[2], weights[2], x, outside)
    for seed in (1, 2):
        x.copy_(randn((m, 256), F16, seed, cuda_device))
        graph.replay()
        torch.cuda.synchronize(cuda_device)
        check(mods[1], weights[1], x, captured)


@pytest.mark.parametrize("m", (1, 40))
def test_weights_and_biases_given_anew(cuda_device, m):
    """A member computes with what it holds, the others as before; copies and modules without their streams stay joined."""
    mods, weights = group(cuda_device)
    x = randn((m, 256), F16, 0, cuda_device)
    for mod, w in zip(mods, weights):
        check(mod, w, x)
    other, u = module(160, 256, 30, cuda_device)
    mods[1].quantized_weights = other.quantized_weights
    mods[2].bias = randn((224,), F16, 31, cuda_device)
    for _ in range(2):
        for mod, w in zip(mods, (weights[0], u, weights[2])):
            check(mod, w, x)
            check(mod, w, x, ab.linear_epilogue(mod, x))
    mods[2].bias = None
    assert_rounded(mods[2](x), *D.product(x, weights[2], None))
    mods, weights = group(cuda_device)
    for mod in mods:
        mod(x)
    for mod in mods:
        mod.offload_canonical()
    for those in (mods, copy.deepcopy(mods)):
        launches = those[0]._group.launches
        for mod, w in zip(those, weights):
            check(mod, w, x)
        assert those[0]._group.launches == launches + 1


@pytest.mark.parametrize("dtype", (F16, torch.float32))
@pytest.mark.parametrize("m", (1, 40))
def test_biases_written_to(cuda_device, m, dtype):
    """In place, alone and in a group: what the kernels read follows, once the write has ended."""
    mods, weights = group(cuda_device)
    x = randn((m, 256), F16, 0, cuda_device)
    for mod in mods:
        mod.bias = mod.bias.to(dtype)
    alone = ab.QuantizedLinear(mods[0].quantized_weights, mods[0].bias)
    for mod, w in zip((*mods, alone), (*weights, weights[0])):
        check(mod, w, x)
    for those in (mods, copy.deepcopy(mods)):
        launches = those[0]._group.launches
        for mod in those:
            mod(x)
        assert those[0]._group.launches == launches + 1
        those[1].bias.add_(1.0)
        those[2].bias.zero_()
        torch.cuda.synchronize(cuda_device)
        for mod, w in zip(those, weights):
            check(mod, w, x)
            check(mod, w, x, ab.linear_epilogue(mod, x))
    late = copy.deepcopy(mods)   # (copied after the writes: what was joined is out of date there too)
    for mod, w in zip(late, weights):
        check(mod, w, x)
    alone.bias.mul_(-2.0)
    torch.cuda.synchronize(cuda_device)
    check(alone, weights[0], x)
    check(alone, weights[0], x, ab.linear_epilogue(alone, x))


@pytest.mark.parametrize("laid_out", (False, True))
def test_first_calls_from_several_threads(cuda_device, laid_out):
    """A group that several threads take into use at once, one of its members laid out before or none."""
    for _ in range(6):
        mods, weights = group(cuda_device)
        if laid_out:
            mods[1]._layout_for(mods[1].quantized_weights)
        inputs = [randn((1 + i, 256), F16, i, cuda_device) for i in range(6)]
        torch.cuda.synchronize(cuda_device)
        outs, errors, start = [None] * len(inputs), [], threading.Barrier(len(inputs))

        def work(i):
            try:
                with torch.cuda.stream(torch.cuda.Stream(cuda_device)):
                    start.wait()
                    if i % 2:
                        outs[i] = [mod(inputs[i]) for mod in mods]
                    else:
                        outs[i] = [ab.linear_epilogue(mod, inputs[i]) for mod in mods]
                    torch.cuda.current_stream(cuda_device).synchronize()
            except BaseException as e:   # noqa: BLE001 - reported by the main thread
                errors.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(inputs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors, errors[0]
        for x, ys in zip(inputs, outs):
            for mod, w, y in zip(mods, weights, ys):
                check(mod, w, x, y)


def test_biases_taken_away(cuda_device):
    """Joined anew without them."""
    mods, weights = group(cuda_device)
    x = randn((2, 256), F16, 0, cuda_device)
    for mod in mods:
        mod(x)
        mod.bias = None
    mods[0]._group.build(x.device)
    for mod, w in zip(mods, weights):
        assert_rounded(mod(x), *D.product(x, w, None))


@pytest.mark.parametrize("m", (1, 12, 40, 200))
def test_biases_that_kernels_in_front_write(cuda_device, m):
    """A bias that another linear's launch is still writing when the module is called with it."""
    long, w = module(1024, 16384, 40, cuda_device, bias=False)
    (lin, v), (up, u) = (module(1024, 256, s, cuda_device) for s in (41, 42))
    x = randn((m, 256), F16, 0, cuda_device)
    for mod in (lin, up):
        mod(x)
    long(randn((1, 16384), F16, 0, cuda_device))
    calls = (lambda: lin(x), lambda: ab.linear_epilogue(lin, x, "relu"), lambda: ab.gated_linear(up, lin, x, "relu"), lambda: ab.gated_linear(lin, up, x, "relu"))
    for seed in range(4):
        for call in calls:
            z = randn((1, 16384), F16, seed, cuda_device)
            torch.cuda.synchronize(cuda_device)
            torch.cuda._sleep(200000)   # (both launches are there before the first one begins)
            lin.bias = long(z)[0]   # (read by the next launch, which need not wait for this one but where it is told to)
            got = call()
            torch.cuda.synchronize(cuda_device)
            assert torch.equal(got, call())
            lin.bias = None
    # in a captured graph: every launch of the call waits for the end of the one in front; later calls need not
    for call in calls:
        lin.bias = None
        ordinary, early = _edges(cuda_device, call, call)
        assert ordinary == 0
        kernels = (early + 1) // 2
        z = randn((1, 16384), F16, 9, cuda_device)

        def front():
            lin.bias = long(z)[0]

        assert _edges(cuda_device, front, call) == (kernels, 0)
        assert _edges(cuda_device, front, lambda: (call(), call())) == (kernels, kernels)
    lin.bias = None


def test_a_group_pickled_without_what_it_joined(cuda_device):
    """As an earlier version of the package wrote it: joined anew at its first call."""
    mods, weights = group(cuda_device)
    x = randn((2, 256), F16, 0, cuda_device)
    for mod in mods:
        mod(x)
    old = mods[0]._group.__getstate__()
    for name in ("_device", "_made_of", "_sizes", "_pieces"):
        del old[name]
    again = object.__new__(type(mods[0]._group))
    again.__setstate__(old)
    for mod in mods:
        mod._group = again
    launches = again.launches
    for mod, w in zip(mods, weights):
        check(mod, w, x)
    assert again.launches == launches + 1
