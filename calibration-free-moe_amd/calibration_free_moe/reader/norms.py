"""The norms before and after a block, fused with its gate and the residual's scale.

A block (attention, a layer of experts) takes the normed residual stream, and its output,
normed again in some models and gated in others, is added to it. `norm_rows` is the first
norm of a stack; `join_block` is all that stands between one block's output and the next
block's input, in one pass over both. The reference leaves these to its host runtime.
"""

from __future__ import annotations

import torch
from torch import Tensor

from calibration_free_moe.reader import _ext

MAX_HIDDEN = 8192
MAX_TOKENS = 2 ** 31 - 1
LARGEST = torch.finfo(torch.float32).max


def _gate_flag(gate: Tensor | None) -> int:
    if gate is None:
        return 0
    if gate.dim() == 1:
        return _ext.GATE_CHANNEL
    return _ext.GATE_ROW if gate.shape[1] == 1 else _ext.GATE_FULL


def _flags(hidden: Tensor, post: Tensor | None, gate: Tensor | None, following: Tensor | None) -> int:
    flags = _gate_flag(gate)
    if hidden.dtype == torch.float32:
        return flags | _ext.FP32
    fp32 = torch.float32
    if post is not None and post.dtype == fp32:
        flags |= _ext.POST_FP32
    if gate is not None and gate.dtype == fp32:
        flags |= _ext.GATE_FP32
    if following is not None and following.dtype == fp32:
        flags |= _ext.NEXT_FP32
    return flags


def _check_hidden(hidden: Tensor, epsilon: float) -> None:
    if (
        hidden.dim() != 2
        or not 1 <= hidden.shape[1] <= MAX_HIDDEN
        or hidden.shape[0] > MAX_TOKENS
        or hidden.dtype not in (torch.bfloat16, torch.float32)
        or not hidden.is_cuda
        or not hidden.is_contiguous()
    ):
        raise ValueError("Expected contiguous BF16 or FP32 CUDA rows [tokens, H], H from 1 to 8192")
    if not isinstance(epsilon, (int, float)) or not 1e-30 <= epsilon <= 1e30:
        raise ValueError("epsilon must be a number between 1e-30 and 1e30")


def _check_weight(weight: Tensor, hidden: Tensor, name: str) -> None:
    if (
        weight.shape != hidden.shape[1:]
        or weight.dtype not in (hidden.dtype, torch.float32)
        or weight.device != hidden.device
        or not weight.is_contiguous()
    ):
        raise ValueError(f"{name} must be contiguous [H] of the rows' type or FP32, on their device")


def norm_rows(hidden: Tensor, weight: Tensor, *, epsilon: float = 1e-6) -> Tensor:
    """hidden / sqrt(mean(hidden^2) + epsilon) * weight, of each row [H] of hidden.

    hidden BF16 or FP32 [tokens, H], H any size from 1 to 8192; weight [H] of that type or
    FP32; epsilon from 1e-30 to 1e30. Sums are FP32, the output is rounded once to the rows'
    type; rows whose squares pass FP32 are scaled first. Gradients go to both, the weight's
    summed over rows in FP32 in an order that depends on sizes alone. One HIP launch on the
    current stream of the rows' device (for the gradient two), which can be captured in a
    graph (a backward pass only where no eager graph of the same leaves is alive).
    """
    _check_hidden(hidden, epsilon)
    _check_weight(weight, hidden, "weight")
    return _ext.operators().join_block(
        hidden, None, None, None, weight, 1.0, epsilon, _flags(hidden, None, None, weight)
    )[0]


def join_block(
    hidden: Tensor,
    block: Tensor,
    *,
    post_weight: Tensor | None = None,
    gate: Tensor | None = None,
    residual_scale: float = 1.0,
    next_weight: Tensor | None = None,
    epsilon: float = 1e-6,
) -> Tensor | tuple[Tensor, Tensor]:
    """joined = residual_scale hidden + gate n, and with `next_weight` (joined, next).

    n is the block's output `block`, or with `post_weight` its norm as of `norm_rows`; next is
    the norm of joined, before joined is rounded, with `next_weight`: what the next block
    takes. hidden and block BF16 or FP32 [tokens, H], of one type; weights [H] of that type or
    FP32; gate, if given, per channel [H] or per row [tokens, 1] of that type or FP32, or
    per value [tokens, H] of that type. H any size from 1 to 8192. residual_scale is a finite
    FP32 number, of the residual stream: one of the block's output is a gate [H] filled with it.

    Gradients go to all tensors, those of weights and of a gate that is spread over rows or
    columns summed in FP32 in an order that depends on sizes alone; they are formed from the
    inputs again, with no other rounding than their own. All inputs are kept for that, and are
    not to change before it. Numbers and launches as `norm_rows`.
    """
    _check_hidden(hidden, epsilon)
    if (
        block.shape != hidden.shape
        or block.dtype != hidden.dtype
        or block.device != hidden.device
        or not block.is_contiguous()
    ):
        raise ValueError("block must be contiguous rows of hidden's shape, type and device")
    if post_weight is not None:
        _check_weight(post_weight, hidden, "post_weight")
    if next_weight is not None:
        _check_weight(next_weight, hidden, "next_weight")
    if gate is not None and (
        gate.shape not in (hidden.shape[1:], (hidden.shape[0], 1), hidden.shape)
        or gate.dtype not in (hidden.dtype, torch.float32)
        or (_gate_flag(gate) == _ext.GATE_FULL and gate.dtype != hidden.dtype)
        or gate.device != hidden.device
        or not gate.is_contiguous()
    ):
        raise ValueError(
            "gate must be contiguous [H] or [tokens, 1] of the rows' type or FP32, or [tokens, H] "
            "of their type, on their device"
        )
    if not isinstance(residual_scale, (int, float)) or not -LARGEST <= residual_scale <= LARGEST:
        raise ValueError("residual_scale must be a finite FP32 number")
    made = _ext.operators().join_block(
        hidden, block, post_weight, gate, next_weight, residual_scale, epsilon,
        _flags(hidden, post_weight, gate, next_weight),
    )
    return made[0] if next_weight is None else tuple(made)


__all__ = ["join_block", "norm_rows"]
