"""The example that runs the linears, the norms and rotations, the cache and the attention together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("generate_with_quantized_cache", os.path.join(ROOT, "examples", "generate_with_quantized_cache.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def prompts_of(lengths, device):
    gen = torch.Generator().manual_seed(4)
    return [torch.randint(0, 1000, (n,), generator=gen).to(device) for n in lengths]


@pytest.mark.parametrize("window,sinks", [(None, 0), (48, 4)])
def test_chunks_and_steps_agree(cuda_device, example, window, sinks):
    """The same tokens through prompts in one piece, in chunks and one by one through the captured step end in the same
    logits: what is cached does not depend on how tokens come, but for roundings of bf16 activations (a few 2^-8 a layer)."""
    prompts = prompts_of((150, 7, 201), cuda_device)
    make = lambda: example.Model(device=cuda_device, window=window, sinks=sinks)  # noqa: E731
    with torch.no_grad():
        whole = make().prefill(prompts, chunk=1000)
        parts = make().prefill(prompts, chunk=64)
        model = make()
        model.prefill([p[:-3] for p in prompts], chunk=100)
        tokens, positions, out, replay = model.decoder()
        for back in (3, 2, 1):
            tokens.copy_(torch.stack([p[-back] for p in prompts]))
            positions.copy_(torch.tensor([len(p) - back for p in prompts], device=cuda_device))
            replay()
        steps = out.clone()
    for other in (parts, steps):
        err = (other.float() - whole.float()).norm(dim=-1) / whole.float().norm(dim=-1)
        assert bool((err < 0.05).all()), err.tolist()


def test_generate(cuda_device, example):
    made, _ = example.generate(example.Model(device=cuda_device), prompts_of((40, 90, 3), cuda_device), 12)
    assert made.shape == (3, 12) and bool((made >= 0).all()) and bool((made < 1000).all())
