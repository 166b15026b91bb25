"""Causal attention with a sliding window and first tokens that stay visible (csrc/kernels/attention.cu), forward and backward.

    out = attention(q, k, v, window=1024, sinks=4)
"""
from __future__ import annotations

import torch

from . import _lib


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int = 0, sinks: int = 0, lengths: torch.Tensor | None = None,
              scale: float | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v over the keys that each query sees, as ``rope_qkv`` lays its parts out: q [batch, tokens, heads, head_dim], k and v
    [batch, tokens, kv_heads, head_dim], bf16, head_dim 64 or 128, heads a multiple of kv_heads (a group of neighbouring heads shares one).

    Query i sees key j where j <= i, and with a ``window`` also i - j < window or j < ``sinks``; ``window`` 0 lets it see all keys up to
    itself.  ``lengths`` (int32 [batch], on the device; numbers beyond [0, tokens] count as the nearest of these) says how many tokens each sequence has: rows behind them are
    zeros in the output and in all gradients, whatever they hold.  ``scale`` is head_dim ** -0.5 unless given.

    Scores, probabilities and sums are computed in 32 bits, the backward pass' probabilities to 7.5e-5; probabilities and their gradients are rounded to bf16 as
    operands of the products, in rows of at most 128 keys to two bf16 each (16 bits together).  For a backward pass the inputs, the output, a byte for each of
    its elements (what rounding it left) and four bytes for each row of a head, in whole 128 rows, are kept.
    Results and gradients are the same bits in every run.  A value in front of a sequence's end that is not finite makes NaN of rows
    that see it.  Products are made of blocks of 128 tokens, in which zero times it is NaN, so it may also of rows up to 512 tokens beyond the window's reach on either
    side, and in dk and dv of blocks that hold sinks.  Tensors may be strided with contiguous heads; where strides or
    addresses are no multiples of 16 bytes they are copied first.  Gradients are of the first order and the reverse mode."""
    return _lib.native().attention(q, k, v, lengths, window, sinks, scale)
