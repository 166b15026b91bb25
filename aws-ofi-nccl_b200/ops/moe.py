"""Tokens sorted by expert and back on one GPU (csrc/kernels/moe_sort.cu): the exchange of a mixture-of-experts layer all of whose
experts are here.  ``parallel.expert_parallel`` moves rows between ranks; these need no communicator and no window, and their order
is that of a stable sort, the same in every run.

Gradients are of the reverse mode; a tensor with a forward-mode tangent is refused.

    order = expert_order(topk_idx, experts)
    rows = permute_tokens(x, order)              # rows [offsets[e], offsets[e + 1]) belong to expert e
    out = unpermute_tokens(y, order, topk_w)     # y: what the experts made of the rows
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class ExpertOrder(NamedTuple):
    """``row_of`` int32 [tokens, k]: the row of each choice, negative (``~row``) for one that goes to no expert; ``offsets`` int32
    [experts + 1]: where each expert's rows begin. Choices without an expert have the rows from ``offsets[-1]`` on."""

    row_of: torch.Tensor
    offsets: torch.Tensor


def expert_order(topk_idx: torch.Tensor, experts: int) -> ExpertOrder:
    """The order of ``topk_idx`` ([tokens, k], int32 or int64) by expert; choices of one expert stay in the order of their tokens.
    Numbers outside [0, experts) go to no expert, which is how padding is left out. Up to 1024 experts."""
    return ExpertOrder(*_lib.native().expert_order(topk_idx, experts))


def permute_tokens(x: torch.Tensor, order: ExpertOrder, scale: torch.Tensor | None = None):
    """x [tokens, H] -> rows [tokens * k, H] in the order of the experts, zeros behind ``offsets[-1]``.  bf16 and fp32 rows have a gradient;
    e4m3 rows have none and take their scales ([tokens] or [tokens, groups], fp32) along, which returns (rows, row_scale)."""
    out = _lib.native().permute_tokens(x, order.row_of, scale)
    return out[0] if scale is None else (out[0], out[1])


def unpermute_tokens(rows: torch.Tensor, order: ExpertOrder, topk_w: torch.Tensor | None = None) -> torch.Tensor:
    """rows [tokens * k, H] (bf16 or fp32) -> [tokens, H], each token's rows summed in 32 bits, weighted by ``topk_w`` (fp32 [tokens, k])
    unless that is None.  Choices without an expert add nothing and their rows are not read.  Rows and weights have gradients, of the
    weighted sum the first ones only."""
    return _lib.native().unpermute_tokens(rows, order.row_of, topk_w)
