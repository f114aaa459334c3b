"""What a decoder step computes around its quantized linears: from the stream of hidden rows to the answer.

The reference leaves these to the model's own modules.

* ``residual_norm``     a block's output normed, gated, scaled and added to the stream, and the sum normed for the next block
* ``linear_epilogue``   a ``QuantizedLinear`` with its activation, scale and residual sum in the same pass
* ``gated_linear``      two of them whose outputs are multiplied, one behind an activation: gate and up of an MLP
* ``token_logprobs``    log probabilities of given tokens, the entropy of every row of logits, and its likeliest tokens

Inference only: no gradients are recorded.  Outputs are computed in fp32 and rounded once, on the current stream of the tensors'
device, and nothing is decided on the host that depends on their contents: it can be captured (linears that have run once before).

The two linears multiply what ``QuantizedLinear`` multiplies, fp16 numbers: bf16 activations become fp16 first, so that those beyond
65504, infinite ones among them, count as 65504 (of their sign; NaN stays NaN) and those below 2^-14 lose bits, down to 2^-25, which
is 0.  The bf16 output of ``gated_linear`` may be larger; ``scale`` there, and its reciprocal in the next linear, keeps it in range.
Residuals and outputs are of the full range.  Both take a module's weight and bias, and go around its forward hooks.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _capi
from .integration.atlas_wrappers import QuantizedLinear, _pending, status_word

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def residual_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                  post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, scale: float = 1.0, eps: float = 1e-6,
                  weight_offset: float = 0.0, centered: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(normed, stream)`` for a block's output ``x`` (``[..., hidden]``, fp16 or bf16, hidden up to 32768)::

        b      = x, or norm(x) * (post_weight + weight_offset)
        stream = residual + scale * gate * b
        normed = norm(stream) * (weight + weight_offset) + bias

    ``norm(v) = v * rsqrt(mean(v^2) + eps)``, or with ``centered`` that of ``v - mean(v)`` (a layer norm); no ``weight`` is 1.
    ``residual`` (of ``x``'s shape) may be fp32, and so is the stream then; without one the stream is the scaled, gated block,
    or ``x`` itself where there is nothing to do.  ``gate`` is ``[hidden]`` or of ``x``'s shape.  Gate, weights and bias are of
    ``x``'s dtype or fp32.  ``normed`` (of ``x``'s dtype) is made of the stream before it is rounded."""
    return _capi.native().residual_norm(x, residual, weight, bias, post_weight, gate, scale, eps, weight_offset, centered)


def _laid_out(linear: QuantizedLinear, device: torch.device):
    """``(layout, bias, whether the bias may still be written)`` of a module on ``device``, as its own forward uses them."""
    if not isinstance(linear, QuantizedLinear):
        raise TypeError(f"expected a QuantizedLinear, got {type(linear)}")
    return linear.kernel_form(device)


def _run(x, first, second, activation, residual, scale):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r} is none of {tuple(ACTIVATIONS)}")
    if not x.is_cuda:
        raise ValueError("x must be on a CUDA device")
    layout, bias, pending = _laid_out(first, x.device)
    pending |= bool(layout.ready) and _pending(layout)
    buffers = lambda l: [l.tiles, l.scales_tiled, l.chunk_ptr, l.entries, l.vals_sorted]  # noqa: E731
    up, up_bias = [], None
    if second is not None:
        other, up_bias, new = _laid_out(second, x.device)
        if (other.n_rows, other.n_cols, other.block_size) != (layout.n_rows, layout.n_cols, layout.block_size):
            raise ValueError(f"gate is [{layout.n_rows}, {layout.n_cols}] in blocks of {layout.block_size}, "
                             f"up [{other.n_rows}, {other.n_cols}] in blocks of {other.block_size}")
        pending |= new | (bool(other.ready) and _pending(other))
        up = buffers(other)
    return _capi.native().fused_linear(x, buffers(layout), bias, up, up_bias, layout.n_rows, layout.n_cols, layout.block_size, residual,
                                       ACTIVATIONS[activation], scale, status_word(x.device), pending)


def linear_epilogue(linear: QuantizedLinear, x: torch.Tensor, activation: Optional[str] = None, *, residual: Optional[torch.Tensor] = None,
                    scale: float = 1.0) -> torch.Tensor:
    """``residual + scale * activation(x W^T + bias)`` of ``linear`` in one pass, rounded once (bf16 activations: see above).

    ``activation``: None, "relu", "silu", "gelu" (by the error function) or "gelu_tanh".  ``residual`` has the result's shape
    and ``x``'s dtype.  ``linear`` may belong to a fused group; only its own rows are computed."""
    return _run(x, linear, None, activation, residual, scale)


def gated_linear(gate: QuantizedLinear, up: QuantizedLinear, x: torch.Tensor, activation: Optional[str] = "silu", *,
                 residual: Optional[torch.Tensor] = None, scale: float = 1.0) -> torch.Tensor:
    """``residual + scale * activation(x G^T + b) * (x U^T + c)`` of ``gate`` and ``up`` in one pass, rounded once; they have one
    shape and block size and may, but need not, be in a fused group.  Arguments as for ``linear_epilogue``."""
    return _run(x, gate, up, activation, residual, scale)


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns."""

    logprobs: torch.Tensor       # fp32, of the tokens' shape
    entropy: torch.Tensor        # fp32, of the tokens' shape
    top_tokens: torch.Tensor     # int64 [..., top], likeliest first
    top_logprobs: torch.Tensor   # fp32 [..., top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities of ``tokens`` (int32 or int64) under ``softmax(logits / temperature)`` (``[..., vocabulary]``, fp16, bf16
    or fp32), the entropy of every row in nats, and its ``top`` (at most 32) likeliest tokens, equal ones by their index.

    A negative token stands for none: its log probability is 0; one beyond the vocabulary gives NaN.  Logits of -inf are tokens
    that cannot follow (log probability -inf); in a row of nothing else all log probabilities are -inf and the entropy is 0.  A
    row with NaN or +inf gives NaN; its top tokens are the largest logits all the same, NaN above them."""
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"token_logprobs: temperature {temperature} is not between 1e-4 and 1e4")
    return TokenLogprobs(*_capi.native().token_logprobs(logits, tokens, top, temperature))
