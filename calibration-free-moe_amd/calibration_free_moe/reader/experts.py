"""The whole routed part of one MoE layer, for a batch of few tokens.

The dense counterpart of a `ProgressiveReader` call over the same borrowed
weights: what a runtime runs for layers that its plan leaves dense, for rows it
does not send to the reader (the reference's runtime sends it decode rows only,
runtime/experts.py:334-378), for an always-on shared expert (one expert, one id),
and as the exact output a sparse one is compared with. With `Fp4Weights` it reads
the experts in 4.25 bits a weight instead of 16. Two to four HIP launches on the
caller's stream (cfmoe_routed_experts in the reader's library). Forward only, as
the reader.
"""

from __future__ import annotations

import torch
from torch import Tensor

from calibration_free_moe.activation import GatedActivation
from calibration_free_moe.reader import _ext
from calibration_free_moe.reader.microscale import Fp4Weights


def routed_experts(
    hidden: Tensor,
    gate_up: Tensor | Fp4Weights,
    down: Tensor | Fp4Weights,
    ids: Tensor,
    weights: Tensor,
    padding: Tensor | None = None,
    out: Tensor | None = None,
    *,
    activation: GatedActivation = "silu",
) -> Tensor:
    """Routed-expert output BF16 [tokens, H]: sum_k w_k D_e (phi(G_e x) * (U_e x)).

    hidden BF16 [tokens, H]; ids (int32/int64) and weights (FP32/BF16) [tokens, K];
    padding bool [tokens] marks rows that read no weights and come out zero.
    gate_up BF16 [E, 2 I, H] and down the channel-major logical [E, H, I] (stride
    (H I, 1, H), the first of one expert whatever it is), as the reader borrows them
    (`channel_major_down`), or both `Fp4Weights` of those logical shapes. Ids outside
    [0, E) contribute nothing; an expert named twice by one token counts twice. Sums are
    FP32, the weighted activations are held to 2^-16, and the output is rounded once.
    Results do not depend on the other tokens of the batch in more than the order of
    FP32 sums. Infinities and NaN stay in the rows that they reach, and an infinite
    weight of `down` makes its output infinite.

    H is a multiple of 128 and I of 16 (of 32 in 4 bits), both at most 4096; at
    most 4096 experts, 64 ids per token and 8192 pairs per call. Zero tokens give
    an empty output; `out` may be `hidden`. The scratch is allocated per call: calls may overlap on
    different streams, and captured graphs share nothing.
    """
    fp4 = isinstance(gate_up, Fp4Weights)
    if fp4 != isinstance(down, Fp4Weights):
        raise ValueError("gate_up and down must both be BF16 tensors or both Fp4Weights")
    if hidden.dim() != 2 or len(gate_up.shape) != 3 or ids.dim() != 2:
        raise ValueError("Expected rows [tokens, H], gate_up [E, 2 I, H] and ids [tokens, K]")
    tokens, h = hidden.shape
    e, rows, _ = gate_up.shape
    i, k = rows // 2, ids.shape[1]
    device = hidden.device
    if (
        gate_up.shape != (e, 2 * i, h)
        or tuple(down.shape) != (e, h, i)
        or not hidden.is_cuda
        or gate_up.device != device
        or down.device != device
        or (fp4 and not (gate_up.valid() and down.valid()))
        or (
            not fp4
            and (
                gate_up.dtype != torch.bfloat16
                or down.dtype != torch.bfloat16
                or not gate_up.is_contiguous()
                or down.stride() != (h * i if e > 1 else down.stride(0), 1, h)
            )
        )
    ):
        raise ValueError(
            "Expected native gate/up [E, 2 I, H] and channel-major down [E, H, I] BF16 CUDA "
            "experts, or Fp4Weights of both"
        )
    if (
        hidden.dtype != torch.bfloat16
        or not hidden.is_contiguous()
        or ids.shape[0] != tokens
        or weights.shape != ids.shape
        or ids.device != device
        or weights.device != device
        or ids.dtype not in (torch.int32, torch.int64)
        or weights.dtype not in (torch.float32, torch.bfloat16)
        or not ids.is_contiguous()
        or not weights.is_contiguous()
        or (
            padding is not None
            and (
                padding.shape != (tokens,)
                or padding.device != device
                or padding.dtype != torch.bool
                or not padding.is_contiguous()
            )
        )
        or (
            out is not None
            and (
                out.shape != hidden.shape
                or out.dtype != hidden.dtype
                or out.device != device
                or not out.is_contiguous()
            )
        )
    ):
        raise ValueError(
            "Expected contiguous BF16 rows, int32/int64 ids, FP32/BF16 weights, bool padding and "
            "BF16 out of one batch on one device"
        )
    if activation not in ("silu", "gelu_tanh"):
        raise ValueError(f"Unsupported routed expert activation: {activation}")
    if out is None:
        out = torch.empty_like(hidden)
    flags = (
        (_ext.IDS_INT64 if ids.dtype == torch.int64 else 0)
        | (_ext.WEIGHTS_BF16 if weights.dtype == torch.bfloat16 else 0)
        | (_ext.GELU if activation == "gelu_tanh" else 0)
        | (_ext.FP4 if fp4 else 0)
    )
    size = _ext.routed_experts_scratch_bytes(h, i, e, k, flags, tokens)
    if not tokens:
        return out
    scratch = torch.empty(size, dtype=torch.uint8, device=device)
    if fp4:
        pointers = (gate_up.codes.data_ptr(), gate_up.scales.data_ptr(), down.codes.data_ptr(),
                    down.scales.data_ptr())
    else:
        pointers = (gate_up.data_ptr(), None, down.data_ptr(), None)
    _ext.run(
        _ext.library().cfmoe_routed_experts, device, h, i, e, k, flags, *pointers,
        hidden.data_ptr(), ids.data_ptr(), weights.data_ptr(),
        None if padding is None else padding.data_ptr(), out.data_ptr(), scratch.data_ptr(),
        tokens,
    )
    return out


__all__ = ["routed_experts"]
