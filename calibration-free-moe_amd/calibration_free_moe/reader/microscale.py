"""Microscaled 4-bit weights (MXFP4): quantisation, values, and their container.

A second way to read fewer bytes of an expert, next to the sketch: every weight
is kept, in 4.25 bits. 32 consecutive values of the last dimension share one E8M0
scale 2^(byte - 127) and are E2M1 numbers (0, .5, 1, 1.5, 2, 3, 4, 6 and their
negatives), the block format of the OCP Microscaling specification. `routed_experts`
multiplies by such weights directly. The reference has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from calibration_free_moe.reader import _ext

# Values that share a scale.
BLOCK = 32


@dataclass(frozen=True)
class Fp4Weights:
    """Microscaled 4-bit weights of logical shape [..., n], n a multiple of 32.

    `codes` uint8 [..., n / 2] holds element 2 i in the low nibble of byte i and
    element 2 i + 1 in the high one, each a sign bit over three bits of E2M1;
    `scales` uint8 [..., n / 32] holds the E8M0 bytes (255 is NaN). Both contiguous.
    """

    codes: Tensor
    scales: Tensor

    @property
    def shape(self) -> torch.Size:
        """The logical shape [..., n]."""
        return torch.Size((*self.codes.shape[:-1], 2 * self.codes.shape[-1]))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def valid(self) -> bool:
        """Whether codes and scales are contiguous bytes of one shape on one GPU."""
        codes, scales = self.codes, self.scales
        return (
            codes.dim() >= 1
            and codes.shape[-1] % (BLOCK // 2) == 0
            and scales.shape == (*codes.shape[:-1], codes.shape[-1] // (BLOCK // 2))
            and codes.dtype == scales.dtype == torch.uint8
            and codes.is_cuda
            and scales.device == codes.device
            and codes.is_contiguous()
            and scales.is_contiguous()
        )


def quantise_fp4(weights: Tensor) -> Fp4Weights:
    """Quantise contiguous BF16 or FP32 weights [..., n] in one HIP launch.

    Per block of 32: the scale is 2^(floor(log2 max|v|) - 2), at least 2^-125, and
    each value / scale is rounded to the nearest E2M1 number, ties to the even
    mantissa; quotients beyond 6 become 6. A block that holds a NaN or an infinity
    gets scale 255 and reads back as NaN. The block runs along the last dimension,
    which is the one a product sums over: give `routed_experts` its down weights
    quantised from a contiguous [E, H, I] (a channel-major view's `.contiguous()`).
    """
    if (
        weights.dim() < 1
        or weights.shape[-1] % BLOCK
        or weights.dtype not in (torch.bfloat16, torch.float32)
        or not weights.is_cuda
        or not weights.is_contiguous()
    ):
        raise ValueError(
            "Expected contiguous BF16 or FP32 CUDA weights whose last dimension is a multiple of 32"
        )
    lead, n = weights.shape[:-1], weights.shape[-1]
    device = weights.device
    codes = torch.empty((*lead, n // 2), dtype=torch.uint8, device=device)
    scales = torch.empty((*lead, n // BLOCK), dtype=torch.uint8, device=device)
    flags = _ext.FP32 if weights.dtype == torch.float32 else 0
    _ext.run(
        _ext.library().cfmoe_quantise_fp4, device, scales.numel(), flags, weights.data_ptr(),
        codes.data_ptr(), scales.data_ptr(),
    )
    return Fp4Weights(codes, scales)


def dequantise_fp4(weights: Fp4Weights) -> Tensor:
    """The BF16 values [..., n] that codes and scales stand for, exactly.

    A scale byte of 254, which `quantise_fp4` never gives, makes magnitudes of 2 and
    more infinite, 255 every value NaN.
    """
    if not weights.valid():
        raise ValueError("Expected contiguous CUDA codes [..., n / 2] and scales [..., n / 32]")
    values = torch.empty(weights.shape, dtype=torch.bfloat16, device=weights.device)
    _ext.run(
        _ext.library().cfmoe_dequantise_fp4, weights.device, weights.scales.numel(),
        weights.codes.data_ptr(), weights.scales.data_ptr(), values.data_ptr(),
    )
    return values


__all__ = ["BLOCK", "Fp4Weights", "dequantise_fp4", "quantise_fp4"]
