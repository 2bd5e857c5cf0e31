"""Tokens laid out by expert, and back, with the router's weights and gradients.

What stands between `route` and products over many rows of one expert (a prompt's
tokens, a training step): the batch's pairs of token and slot are sorted by expert,
`gather_rows` lays out a row for each, the caller's products take the rows of expert e,
`offsets[e]` to `offsets[e + 1]`, and `combine_rows` sums what they give. The reference
has no counterpart; its operator takes the router's ids and weights as they are
(calibration_free_moe/reader/progressive.py:3876-3885).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from calibration_free_moe.reader import _ext

MAX_HIDDEN = 1 << 20
MAX_EXPERTS = 4096
MAX_TOP_K = 64
MAX_PAIRS = 1 << 30


@dataclass(frozen=True)
class ExpertOrder:
    """A batch's pairs in expert order, all int32 on one GPU (`sort_by_expert` makes it).

    Rows are the kept pairs by expert, those of one expert in the batch's order, and
    behind them the dropped pairs. `offsets` [E + 1]: expert e has the rows from
    offsets[e] to offsets[e + 1], and offsets[E] rows are kept. `places` [tokens, K]: the
    row of each pair, or -1 - row of a dropped one. `pairs` [tokens K]: t K + k of each row.
    """

    offsets: Tensor
    places: Tensor
    pairs: Tensor

    def __post_init__(self) -> None:
        offsets, places, pairs = self.offsets, self.places, self.pairs
        if (
            places.dim() != 2
            or not 1 <= places.shape[1] <= MAX_TOP_K
            or offsets.dim() != 1
            or pairs.dim() != 1
            or offsets.shape[0] < 2
            or pairs.shape[0] != places.numel()
            or places.numel() > MAX_PAIRS
            or not offsets.dtype == places.dtype == pairs.dtype == torch.int32
            or not offsets.device == places.device == pairs.device
            or not places.is_contiguous()
            or not pairs.is_contiguous()
            or not offsets.is_contiguous()
        ):
            raise ValueError("Expected contiguous int32 tensors of one batch for an ExpertOrder")


def sort_by_expert(ids: Tensor, experts: int, padding: Tensor | None = None) -> ExpertOrder:
    """The order of a batch's pairs by expert, from `route`'s ids (int32/int64) [tokens, K].

    A pair is kept where its id lies in [0, experts) and its token is not marked in
    `padding` (bool [tokens]); the others (experts of another GPU, a batch padded to its
    capture size) are dropped and sorted behind. The sort is stable, and its integers are
    the same for every call. At most 4096 experts, 64 ids per token and 2^30 pairs. Zero
    tokens give an empty order. One or two HIP launches on the current stream of the ids'
    device, which the host does not wait for; they can be captured in a graph.
    """
    if (
        ids.dim() != 2
        or ids.dtype not in (torch.int32, torch.int64)
        or not ids.is_cuda
        or not ids.is_contiguous()
    ):
        raise ValueError("Expected contiguous int32 or int64 CUDA ids [tokens, K]")
    tokens, top_k = ids.shape
    device = ids.device
    if not 1 <= experts <= MAX_EXPERTS or not 1 <= top_k <= MAX_TOP_K or ids.numel() > MAX_PAIRS:
        raise ValueError("Expected 1 to 4096 experts, 1 to 64 ids per token and at most 2^30 pairs")
    if padding is not None and (
        padding.shape != (tokens,)
        or padding.device != device
        or padding.dtype != torch.bool
        or not padding.is_contiguous()
    ):
        raise ValueError("padding must be contiguous bool [tokens] on the ids' device")
    offsets, places, pairs = _ext.operators().sort_by_expert(ids, experts, padding)
    # (as made here the three need no check)
    order = ExpertOrder.__new__(ExpertOrder)
    order.__dict__.update(offsets=offsets, places=places, pairs=pairs)
    return order


def _check_rows(rows: Tensor, count: int, order: ExpertOrder, what: str) -> None:
    if (
        rows.dim() != 2
        or rows.shape[0] != count
        or not 1 <= rows.shape[1] <= MAX_HIDDEN
        or rows.dtype not in (torch.bfloat16, torch.float32)
        or not rows.is_cuda
        or rows.device != order.places.device
        or not rows.is_contiguous()
    ):
        raise ValueError(
            f"Expected contiguous BF16 or FP32 CUDA {what} of the order's batch on its GPU, "
            "H from 1 to 2^20"
        )


def gather_rows(hidden: Tensor, order: ExpertOrder) -> Tensor:
    """Rows [tokens K, H] of the order's pairs, from hidden (BF16 or FP32) [tokens, H].

    Row r is hidden[order.pairs[r] // K]; rows of dropped pairs are zero. The gradient of
    hidden is the sum of its kept pairs' row gradients in slot order, in FP32, rounded once;
    gradients of dropped rows are not read. H is any size from 1 to 2^20. One HIP launch on
    the current stream of the rows' device, for the gradient another; both can be captured
    in a graph (a backward pass only where no eager graph of the same leaves is alive).
    """
    _check_rows(hidden, order.places.shape[0], order, "rows [tokens, H]")
    return _ext.operators().gather_rows(hidden, order.places)


def combine_rows(rows: Tensor, order: ExpertOrder, weights: Tensor | None = None) -> Tensor:
    """out [tokens, H]: each token's kept rows, times its weights, summed in slot order.

    rows (BF16 or FP32) [tokens K, H] in the order's rows, weights (FP32 or BF16)
    [tokens, K] as `route` gives them, or None for ones. Sums are FP32, rounded once to the
    rows' type; what a dropped pair's row and weight hold is not read, and a token without
    a kept pair gives zeros. Gradients go to rows (zero in dropped rows) and weights (the
    FP32 sum of out's gradient times the row; zero for dropped pairs). Launches as
    `gather_rows`.
    """
    places = order.places
    _check_rows(rows, places.numel(), order, "rows [tokens K, H]")
    if weights is not None and (
        weights.shape != places.shape
        or weights.dtype not in (torch.float32, torch.bfloat16)
        or weights.device != places.device
        or not weights.is_contiguous()
    ):
        raise ValueError("weights must be contiguous FP32 or BF16 [tokens, K] on the rows' device")
    return _ext.operators().combine_rows(rows, places, weights)


__all__ = ["ExpertOrder", "combine_rows", "gather_rows", "sort_by_expert"]
