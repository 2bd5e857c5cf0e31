"""Low-rank adapters of a batch's requests beside a projection that they share.

Requests of one batch may each bring an adapter of their own for a projection (a shared
expert's gate, up or down rows, a router, the projections of attention): the projection's
product is made once for all of them, and `apply_adapters` adds each token's low-rank
product to it, whatever mixture of adapters the batch holds. Forward only, as the reader.
The reference's own low-rank map, its recovery bank, is one for all tokens
(calibration_free_moe/reader/progressive.py:1859-2016).
"""

from __future__ import annotations

import torch
from torch import Tensor

from calibration_free_moe.reader import _ext

MAX_SIZE = 65536
MAX_RANK = 256
MAX_ADAPTERS = 4096
MAX_TOKENS = 1 << 24


def _stride(t: Tensor) -> int:
    """Values from one row to the next; of a single row, which has none, its length."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _rows(t: Tensor, device: torch.device) -> bool:
    """Whether t is BF16 rows on the device, of consecutive values, 16-byte aligned."""
    step, one = t.stride()
    return (
        t.dtype == torch.bfloat16
        and t.device == device
        and one == 1
        and (step % 8 == 0 or t.shape[0] < 2)
        and t.data_ptr() % 16 == 0
    )


def _overlap(out: Tensor, rows: Tensor) -> bool:
    """Whether two of a call's rows share memory and are not the same rows."""
    if out.shape == rows.shape and out.data_ptr() == rows.data_ptr() and _stride(out) == _stride(rows):
        return False
    tokens, step = out.shape[0], _stride(out)
    ends = [t.data_ptr() + 2 * ((tokens - 1) * _stride(t) + t.shape[1]) for t in (out, rows)]
    if ends[0] <= rows.data_ptr() or ends[1] <= out.data_ptr():
        return False
    # columns of one wide tensor lie between each other's and share nothing
    apart = (rows.data_ptr() - out.data_ptr()) // 2 % step
    return (
        tokens == 1
        or _stride(rows) != step
        or apart < out.shape[1]
        or apart + rows.shape[1] > step
    )


def apply_adapters(
    base: Tensor,
    hidden: Tensor,
    encoder: Tensor,
    decoder: Tensor,
    slots: Tensor,
    scales: Tensor | None = None,
    out: Tensor | None = None,
) -> Tensor:
    """out[t] = base[t] + scales[a] decoder[a] (encoder[a] hidden[t]), a = slots[t].

    base BF16 [tokens, O] is the shared projection's product of hidden BF16 [tokens, H];
    encoder BF16 [N, R, H] and decoder BF16 [N, O, R] hold N adapters of rank R (one of lower
    rank with zeros behind), contiguous; slots (int32/int64) [tokens] names each token's
    adapter, and a slot outside [0, N) none: its row comes out as it is in base, bit for bit.
    scales FP32 [N], or None for ones. Sums are FP32, the R inner values are held in
    FP32's 24 bits, and the output is rounded once.

    base, hidden and out may be column slices of wider rows (first stride a multiple of 8,
    16-byte aligned). `out` may be `base`, whose rows without an adapter are then left
    alone, or `hidden`; no other overlap. H and O are multiples of 8 up to 65536, R of 8 up
    to 256, N up to 4096, tokens up to 2^24; zero tokens give an empty output. One or two HIP
    launches on the current stream of the tensors' device, up to four for more than 256 tokens,
    with scratch allocated per call where they need any; they can be captured in a graph. `out`
    counts as written in place. Tensors that require gradients, `out` among them, are refused
    while gradients are on.
    """
    if hidden.dim() != 2 or base.dim() != 2 or encoder.dim() != 3 or decoder.dim() != 3:
        raise ValueError(
            "Expected base [tokens, O], hidden [tokens, H], encoder [N, R, H] and decoder [N, O, R]"
        )
    tokens, h = hidden.shape
    n, rank, encoded = encoder.shape
    device = hidden.device
    o = base.shape[1]
    if (
        h % 8
        or not 8 <= h <= MAX_SIZE
        or o % 8
        or not 8 <= o <= MAX_SIZE
        or rank % 8
        or not 8 <= rank <= MAX_RANK
        or not 1 <= n <= MAX_ADAPTERS
        or tokens > MAX_TOKENS
    ):
        raise ValueError(
            "Expected hidden and output sizes that are multiples of 8 up to 65536, a rank that is "
            "one up to 256, 1 to 4096 adapters and at most 2^24 tokens"
        )
    if (
        encoded != h
        or decoder.shape != (n, o, rank)
        or base.shape[0] != tokens
        or not hidden.is_cuda
        or encoder.dtype != torch.bfloat16
        or decoder.dtype != torch.bfloat16
        or encoder.device != device
        or decoder.device != device
        or not encoder.is_contiguous()
        or not decoder.is_contiguous()
        or not _rows(hidden, device)
        or not _rows(base, device)
    ):
        raise ValueError(
            "Expected BF16 CUDA rows [tokens, H] and [tokens, O], 16-byte aligned with a first "
            "stride of a multiple of 8, and contiguous BF16 encoder [N, R, H] and decoder [N, O, R]"
        )
    if (
        slots.shape != (tokens,)
        or slots.dtype not in (torch.int32, torch.int64)
        or slots.device != device
        or not slots.is_contiguous()
        or (
            scales is not None
            and (
                scales.shape != (n,)
                or scales.dtype != torch.float32
                or scales.device != device
                or not scales.is_contiguous()
            )
        )
    ):
        raise ValueError(
            "Expected contiguous int32/int64 slots [tokens] and FP32 scales [N] on the rows' device"
        )
    if torch.is_grad_enabled() and (
        base.requires_grad
        or hidden.requires_grad
        or encoder.requires_grad
        or decoder.requires_grad
        or (scales is not None and scales.requires_grad)
        or (out is not None and out.requires_grad)
    ):
        raise ValueError(
            "apply_adapters is forward only: detach its inputs and out or call it in no_grad"
        )
    if out is not None:
        if out.shape != base.shape or not _rows(out, device) or _stride(out) < o:
            raise ValueError(
                "out must be BF16 rows [tokens, O] on the rows' device, one behind another"
            )
        if tokens and (_overlap(out, base) or _overlap(out, hidden)):
            raise ValueError("out overlaps base or hidden and is not the same rows")
    return _ext.operators().apply_adapters(base, hidden, encoder, decoder, slots, scales, out)


__all__ = ["apply_adapters"]
