"""A decoder with quantized linears and a 4-bit key/value cache, end to end: prompts of different lengths, then tokens.

    python examples/generate_with_quantized_cache.py [--layers 4 --hidden 1024 --tokens 32]

Random weights of a Llama pattern (grouped queries, norms on queries and keys).  The prompts go through the layers as one
ragged batch, in chunks; the tokens after them one step at a time, captured once as a CUDA graph and replayed, since nothing
about lengths or pages is decided on the host.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import atlasinfer_b200 as ab  # noqa: E402

DTYPE = torch.bfloat16


class Layer:
    """Attention and MLP of one layer; its weights quantized, its keys and values in a cache of its own."""

    def __init__(self, hidden, heads, kv_heads, head_dim, pages, page_size, device, gen, window=None, sinks=0):
        self.heads, self.kv_heads, self.head_dim, self.window, self.sinks = heads, kv_heads, head_dim, window, sinks
        inter = 2 * hidden
        shapes = [(heads * head_dim, hidden), (kv_heads * head_dim, hidden), (kv_heads * head_dim, hidden), (hidden, heads * head_dim),
                  (inter, hidden), (inter, hidden), (hidden, inter)]
        weights = [(torch.randn(n, k, generator=gen, device=device) * k ** -0.5).half() for n, k in shapes]
        self.q, self.k, self.v, self.o, self.gate, self.up, self.down = (ab.QuantizedLinear(w, None) for w in ab.quantize_tensors(weights))
        self.groups = [ab.fuse_linears([self.q, self.k, self.v]), ab.fuse_linears([self.gate, self.up])]
        self.q_norm, self.k_norm = (1 + 0.1 * torch.randn(2, head_dim, generator=gen, device=device)).to(DTYPE)
        self.cache = ab.QuantizedKVCache(pages, kv_heads, head_dim, page_size=page_size, device=device)

    def __call__(self, x, step):
        h = torch.nn.functional.rms_norm(x, x.shape[-1:])
        q, k, v = (m(h).unflatten(-1, (-1, self.head_dim)) for m in (self.q, self.k, self.v))
        q = ab.norm_rotate_store(q, k, v, self.cache, step["slots"], step["table"], step["positions"], q_weight=self.q_norm, k_weight=self.k_norm)
        a = ab.cache_attention(q, self.cache, step["pages"], step["lengths"], query_starts=step["starts"], max_queries=step["most"],
                               window=self.window, sinks=self.sinks)
        x = x + self.o(a.flatten(1))
        h = torch.nn.functional.rms_norm(x, x.shape[-1:])
        return x + self.down(torch.nn.functional.silu(self.gate(h)) * self.up(h))


class Model:
    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, vocab=1000, sequences=3, context=512, page_size=32, device="cuda", seed=0,
                 window=None, sinks=0):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.device, self.page_size, self.sequences = torch.device(device), page_size, sequences
        per = -(-context // page_size)
        # every sequence's pages, shuffled over the pool
        self.pages = torch.randperm(sequences * per, generator=gen, device=device).int().view(sequences, per)
        self.table = ab.rotary_table(context, head_dim, device=device)
        self.every = torch.arange(sequences, device=device)   # (read by the captured step: it has to live as long as the model)
        self.layers = [Layer(hidden, heads, kv_heads, head_dim, sequences * per, page_size, device, gen, window, sinks) for _ in range(layers)]
        self.embedding = torch.randn(vocab, hidden, generator=gen, device=device).to(DTYPE)

    def _slots(self, sequence, positions):
        return self.pages[sequence, positions // self.page_size].long() * self.page_size + positions % self.page_size

    def forward(self, tokens, step):
        x = self.embedding[tokens]
        for layer in self.layers:
            x = layer(x, step)
        return torch.nn.functional.rms_norm(x, x.shape[-1:]) @ self.embedding.T

    def prefill(self, prompts, chunk=256):
        """The logits behind every prompt's last token; the prompts go through in chunks, as ragged batches."""
        last = [None] * len(prompts)
        for at in range(0, max(len(p) for p in prompts), chunk):
            parts = [p[at:at + chunk] for p in prompts]
            counts = [len(p) for p in parts]
            positions = torch.cat([torch.arange(at, at + n, device=self.device) for n in counts])
            sequence = torch.repeat_interleave(torch.arange(len(parts), device=self.device), torch.tensor(counts, device=self.device))
            starts = torch.tensor([0] + counts, dtype=torch.int32, device=self.device).cumsum(0, dtype=torch.int32)
            lengths = torch.tensor([at + n if n else 0 for n in counts], dtype=torch.int32, device=self.device)
            step = dict(slots=self._slots(sequence, positions), table=self.table, positions=positions, pages=self.pages, lengths=lengths, starts=starts,
                        most=max(counts))
            logits = self.forward(torch.cat(parts), step)
            for i, n in enumerate(counts):
                if n:
                    last[i] = logits[int(starts[i + 1]) - 1]
        return torch.stack(last)

    def decoder(self):
        """A captured step: ``(tokens, positions, logits, replay)``; fill the first two, replay, read the third."""
        tokens = torch.zeros(self.sequences, dtype=torch.long, device=self.device)
        positions = torch.zeros(self.sequences, dtype=torch.long, device=self.device)

        def run():
            step = dict(slots=self._slots(self.every, positions), table=self.table, positions=positions, pages=self.pages, lengths=(positions + 1).int(), starts=None, most=1)
            return self.forward(tokens, step)

        side = torch.cuda.Stream(self.device)   # the first pass lays weights out, which a capture must not
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):
            kept = [layer.cache.data.clone() for layer in self.layers]
            run()
            for layer, data in zip(self.layers, kept):   # (it stored at position 0)
                layer.cache.data.copy_(data)
        torch.cuda.current_stream(self.device).wait_stream(side)
        torch.cuda.synchronize(self.device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = run()
        return tokens, positions, logits, graph.replay


@torch.no_grad()
def generate(model, prompts, count):
    """Greedy tokens behind every prompt, and the seconds that the steps took."""
    logits = model.prefill(prompts)
    tokens, positions, out, replay = model.decoder()
    positions.copy_(torch.tensor([len(p) for p in prompts], device=model.device))
    tokens.copy_(logits.argmax(-1))
    made = [tokens.clone()]
    torch.cuda.synchronize(model.device)
    began = time.perf_counter()
    for _ in range(count - 1):
        replay()
        tokens.copy_(out.argmax(-1))
        positions.add_(1)
        made.append(tokens.clone())
    torch.cuda.synchronize(model.device)
    return torch.stack(made, 1), time.perf_counter() - began


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--tokens", type=int, default=32)
    args = ap.parse_args()
    heads = args.hidden // 64
    model = Model(layers=args.layers, hidden=args.hidden, heads=heads, kv_heads=max(1, heads // 4), sequences=3, context=2048)
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=gen, device="cuda") for n in (700, 33, 1500)]
    made, seconds = generate(model, prompts, args.tokens)
    used = sum(layer.cache.data.numel() for layer in model.layers)
    print(made[:, :12].tolist())
    print(f"{args.tokens - 1} steps of {len(prompts)} sequences in {seconds * 1e3:.1f} ms; caches {used / 1e6:.1f} MB")


if __name__ == "__main__":
    main()
