"""Router of one MoE layer: hidden rows to the expert ids and weights a reader takes.

The reference leaves routing to its host runtime, whose outputs its operator
takes (calibration_free_moe/reader/progressive.py:3876-3885). Here `route` makes
them on the caller's stream in two HIP launches (cfmoe_route in the reader's
library), so that a layer is `route` followed by a `ProgressiveReader` call or by
`routed_experts`. Forward only, as the reader.
"""

from __future__ import annotations

import torch
from torch import Tensor

from calibration_free_moe.reader import _ext

MAX_HIDDEN = 65536
MAX_EXPERTS = 1024
MAX_TOP_K = 64


def route(
    hidden: Tensor,
    router: Tensor,
    top_k: int,
    *,
    renormalise: bool = True,
    expert_scale: Tensor | None = None,
    ids_dtype: torch.dtype = torch.int32,
    weights_dtype: torch.dtype = torch.float32,
    out: tuple[Tensor, Tensor] | None = None,
) -> tuple[Tensor, Tensor]:
    """Return (ids, weights), both [tokens, top_k], of a softmax top-k router.

    hidden BF16 [tokens, H] and router BF16 [E, H], contiguous; the logits are
    hidden @ router.T. Each token's `top_k` largest logits are kept, largest
    first: equal logits go to the lowest expert, NaN counts as the largest, and
    the order is that of the exact logits, not of their FP32 sums (those whose order
    FP32 leaves open are formed again in FP64). Weights are the softmax over the kept
    experts (`renormalise`) or the kept part of the softmax over all, times
    `expert_scale` (FP32 [E]) at each kept expert if it is given; they come from the
    FP32 sums, or the FP64 ones where there are any, finite logits beyond FP32 among
    them. Ids are always distinct and inside [0, E), whatever the rows hold.

    `out` takes (ids, weights) to write instead of new tensors; their types then
    stand for `ids_dtype` (int32 or int64) and `weights_dtype` (FP32 or BF16).
    H is a multiple of 128, at most 65536, E at most 1024, top_k at most 64 and E, and
    there are fewer than 2^21 tiles of 16 tokens by 16 experts. 64 kept of more experts
    form all kept logits in FP64, which takes up to three times as long as 63.
    Zero tokens give empty outputs. The work is enqueued on the current stream of the
    tensors' device and can be captured in a graph.
    """
    if out is not None:
        ids, weights = out
        ids_dtype, weights_dtype = ids.dtype, weights.dtype
    if (
        hidden.dim() != 2
        or router.dim() != 2
        or hidden.shape[1] != router.shape[1]
        or hidden.shape[1] % 128
        or not 0 < hidden.shape[1] <= MAX_HIDDEN
        or not 1 <= router.shape[0] <= MAX_EXPERTS
        or not 1 <= top_k <= min(MAX_TOP_K, router.shape[0])
        or hidden.dtype != torch.bfloat16
        or router.dtype != torch.bfloat16
        or not hidden.is_cuda
        or router.device != hidden.device
        or not hidden.is_contiguous()
        or not router.is_contiguous()
        or ids_dtype not in (torch.int32, torch.int64)
        or weights_dtype not in (torch.float32, torch.bfloat16)
    ):
        raise ValueError(
            "Expected contiguous BF16 CUDA rows [tokens, H] and router [E, H] with H a multiple "
            "of 128 up to 65536, at most 1024 experts and 64 kept, int32/int64 ids and FP32/BF16 weights"
        )
    tokens, experts, device = hidden.shape[0], router.shape[0], hidden.device
    if expert_scale is not None and (
        expert_scale.shape != (experts,)
        or expert_scale.dtype != torch.float32
        or expert_scale.device != device
        or not expert_scale.is_contiguous()
    ):
        raise ValueError("expert_scale must be contiguous FP32 [E] on the router's device")
    if out is None:
        ids = torch.empty((tokens, top_k), dtype=ids_dtype, device=device)
        weights = torch.empty((tokens, top_k), dtype=weights_dtype, device=device)
    elif any(
        t.shape != (tokens, top_k) or t.device != device or not t.is_contiguous() for t in out
    ):
        raise ValueError("out must be contiguous (ids, weights) [tokens, top_k] on the rows' device")
    if not tokens:
        return ids, weights
    flags = (
        (_ext.IDS_INT64 if ids_dtype == torch.int64 else 0)
        | (_ext.WEIGHTS_BF16 if weights_dtype == torch.bfloat16 else 0)
        | (_ext.RENORMALISE if renormalise else 0)
    )
    scratch = torch.empty(
        _ext.route_scratch_bytes(tokens, experts), dtype=torch.uint8, device=device
    )
    _ext.run(
        _ext.library().cfmoe_route, device, hidden.shape[1], experts, top_k, flags,
        hidden.data_ptr(), router.data_ptr(),
        None if expert_scale is None else expert_scale.data_ptr(), ids.data_ptr(),
        weights.data_ptr(), scratch.data_ptr(), tokens,
    )
    return ids, weights


__all__ = ["route"]
