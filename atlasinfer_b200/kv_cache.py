"""Queries, keys and a key/value cache in 4 bits: what a decoder layer does between its quantized linears.

The reference leaves attention to the model and tiers an fp16 cache over GPU, CPU and disk; here the cache stays on the GPU in a
quarter of the memory, and attention reads it as it is.

* ``norm_rotate``        norms of queries and keys for each head, and their position rotation, in one pass
* ``QuantizedKVCache``   pages of keys and values in 4 bits; ``store`` and ``load`` by slot
* ``norm_rotate_store``  ``norm_rotate`` with keys and values written to the cache in the same pass
* ``cache_attention``    attention over the cache: causal, with a sliding window and first tokens that stay visible

Inference only: no gradients are recorded.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _capi
from .integration.atlas_wrappers import status_word

HEAD_DIMS = (64, 128, 256)
SLAB_TOKENS = 16


def rotary_table(max_positions: int, rotary_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """Cosines, then sines, of the angles ``position * base^(-2 i / rotary_dim)``: fp32 ``[max_positions, rotary_dim]``.

    Made in 64 bits, so that far positions keep their angles.  Models that stretch their angles make a table of their own."""
    if rotary_dim < 16 or rotary_dim % 16:
        raise ValueError(f"rotary_dim {rotary_dim} is not a multiple of 16")
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], -1).float()


class QuantizedKVCache:
    """Pages of keys and values of one layer, 4.5 bits a number.

    A page holds ``page_size`` tokens (a multiple of 16) of ``kv_heads`` heads; a token's place is its slot,
    ``page * page_size + offset``, and which pages are whose is the caller's business.  Every 64 channels of a token and
    head share an fp16 scale and a zero point: value ``s * (c - z)``, ``c`` and ``z`` in 0..15, exact in fp16, at most half a
    step from the number stored, where a step is a fifteenth of the range of the 64 (zero included), rounded up to 7 bits.
    That holds for ranges up to 65280, as far as fp16 reaches to one side.  A step is never more than 4352, so 64 numbers of
    both signs that lie further apart keep their low end, and what is more than ``4352 * (15 - z)`` is stored as that, which may
    be far off (60000 beside -60000 as 4352): scale such keys or values down.  NaN is stored as 0, and what passes 65280 to
    either side counts as that, so the cache holds finite numbers only.

    ``data``: storage to use (uint8 ``[num_pages, kv_heads, page_bytes]``, contiguous); default: zero-filled."""

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device=None, data: Optional[torch.Tensor] = None):
        if head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"QuantizedKVCache: head_dim {head_dim} is not one of {HEAD_DIMS}")
        if page_size < SLAB_TOKENS or page_size % SLAB_TOKENS or page_size > 1 << 20:
            raise NotImplementedError(f"QuantizedKVCache: page_size {page_size} is not a multiple of {SLAB_TOKENS} up to 2^20")
        if num_pages < 0 or kv_heads < 1:
            raise ValueError(f"QuantizedKVCache: {num_pages} pages of {kv_heads} heads")
        self.num_pages, self.kv_heads, self.head_dim, self.page_size = int(num_pages), int(kv_heads), int(head_dim), int(page_size)
        shape = (self.num_pages, self.kv_heads, self.page_bytes(head_dim, page_size))
        if data is None:
            data = torch.zeros(shape, dtype=torch.uint8, device=_capi.require_cuda(torch.device(device) if device is not None else None))
        elif data.dtype is not torch.uint8:
            raise TypeError(f"QuantizedKVCache: data must be uint8, got {data.dtype}")
        elif tuple(data.shape) != shape or not data.is_contiguous() or data.data_ptr() % 16:
            raise ValueError(f"QuantizedKVCache: data must be contiguous and {shape}, got {tuple(data.shape)}")
        elif data.device.type != "cuda":
            raise ValueError("QuantizedKVCache: data must be on a CUDA device")
        self.data = data

    @staticmethod
    def page_bytes(head_dim: int, page_size: int) -> int:
        """Bytes of a page for one head."""
        return page_size // SLAB_TOKENS * 18 * head_dim

    @property
    def num_slots(self) -> int:
        return self.num_pages * self.page_size

    @property
    def device(self) -> torch.device:
        return self.data.device

    def store(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Write ``k`` and ``v`` (``[tokens, kv_heads, head_dim]``, fp16 or bf16) to ``slots`` (int32 or int64).

        Tokens whose slot is not in the cache (-1 for padding) are not stored.  A slot may occur once."""
        _capi.native().norm_rotate(None, k, v, None, None, None, None, 0.0, 0.0, False, self.data, self.head_dim, self.page_size, slots)

    def load(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of ``slots`` as ``[tokens, kv_heads, head_dim]``; fp16 is what is stored, bf16 rounds it.

        Slots that are not in the cache give zeros."""
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"QuantizedKVCache.load: dtype must be fp16 or bf16, got {dtype}")
        return _capi.native().kv_load(self.data, self.head_dim, self.page_size, slots, dtype is torch.bfloat16)


def norm_rotate(q: torch.Tensor, k: torch.Tensor, table: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, *,
                q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                weight_offset: float = 0.0, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normed and rotated copies of ``q`` and ``k`` (``[tokens, heads, head_dim]``, fp16 or bf16, any strides).

    With a weight a head becomes ``x * rsqrt(mean(x^2) + eps) * (weight + weight_offset)`` (weights ``[head_dim]``, of the
    tensors' dtype or fp32).  With a ``table`` (``rotary_table``) and ``positions`` (``[tokens]``, int32 or int64) its first
    ``table.shape[1]`` channels are rotated, in pairs half of them apart or (``interleaved``) next to each other.  Computed in
    fp32, rounded once.  The rotated channels of a token whose position is not in the table become NaN."""
    return _capi.native().norm_rotate(q, k, None, table, positions, q_weight, k_weight, eps, weight_offset, interleaved, None, 0, 0, None)


def norm_rotate_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: QuantizedKVCache, slots: torch.Tensor,
                      table: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, *,
                      q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                      weight_offset: float = 0.0, interleaved: bool = False) -> torch.Tensor:
    """``norm_rotate`` whose keys, with ``v``, go to ``slots`` of ``cache`` (as by ``QuantizedKVCache.store``, but without a
    rounding to 16 bits in between); returns the queries.

    The cache holds no NaN: of a token whose position is not in the table, the key's rotated channels are stored as zeros, and
    only its query shows it."""
    return _capi.native().norm_rotate(q, k, v, table, positions, q_weight, k_weight, eps, weight_offset, interleaved,
                                      cache.data, cache.head_dim, cache.page_size, slots)[0]


def cache_attention(q: torch.Tensor, cache: QuantizedKVCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
                    query_starts: Optional[torch.Tensor] = None, max_queries: Optional[int] = None, window: Optional[int] = None,
                    sinks: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of ``q`` (``[queries, heads, head_dim]``, fp16 or bf16) over the cache; heads share kv heads in groups.

    Sequence ``b`` has ``lengths[b]`` tokens (int32) in the pages ``page_table[b]`` (int32 ``[sequences, pages]``); the last
    of them are those of its own queries, which must have been stored.  Its queries are rows ``query_starts[b]`` to
    ``query_starts[b + 1]`` of ``q`` (int32 ``[sequences + 1]``; default: equally many each), at most ``max_queries`` (on the
    host: it decides which kernel runs and how many rows; default: all).  Rows that belong to no sequence, or to one beyond its
    first ``max_queries``, give zeros.  A query sees the keys up to its own position, with a ``window`` only the
    last ``window`` of those and the first ``sinks``; pages that no query sees are not read, and their entries in
    ``page_table`` may be anything.  A query that sees nothing gives zeros.  ``scale`` defaults to ``head_dim ** -0.5``.

    Everything about lengths stays on the device: the call can be captured, and replayed for other lengths."""
    if window is not None and window < 1:
        raise ValueError(f"cache_attention: window {window}")
    if max_queries is not None and max_queries < 0:
        raise ValueError(f"cache_attention: max_queries {max_queries}")
    return _capi.native().kv_attention(q, cache.data, cache.head_dim, cache.page_size, page_table, lengths, query_starts,
                                       -1 if max_queries is None else max_queries, window or 0, sinks,
                                       cache.head_dim ** -0.5 if scale is None else scale, status_word(q.device))
