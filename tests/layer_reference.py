"""Plain 64-bit forms of the router, the whole MoE layer and 4-bit weights (CPU).

Each comes with an element-wise bound on what a right FP32 / matrix-core
computation may be off, from the operands themselves:

* A sum of n products whose additions each round (or cut off) by at most 2^-23 of
  a partial sum is within n_add 2^-23 sum|products| of the exact one, n_add the
  longest chain of additions a term goes through. A matrix instruction adds 32
  products and one accumulator; n / 32 instructions follow one another, and at
  most 64 partial sums (waves, splits, slots, lanes) are added at the end.
* One rounding to BF16 is off by at most 2^-8 of the value (half of eps).
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

STEP = 2.0 ** -23
HALF_BF16 = torch.finfo(torch.bfloat16).eps / 2


def chain(products: int) -> float:
    """n_add 2^-23 for a sum of `products` terms."""
    return (products / 32 + 1 + 33 + 64) * STEP


def phi(gate: Tensor, activation: str) -> Tensor:
    if activation == "silu":
        return gate * torch.sigmoid(gate)
    inner = math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
    return 0.5 * gate * (1 + torch.tanh(inner))


def layer(x: Tensor, gate_up: Tensor, down: Tensor, ids: Tensor, weights: Tensor,
          padding: Tensor | None = None, activation: str = "silu") -> tuple[Tensor, Tensor]:
    """(out, bound) in float64: gate_up [E, 2 I, H], down logical [E, H, I]."""
    tokens, hidden = x.shape
    experts, width = down.shape[0], down.shape[2]
    x, weights = x.double().cpu(), weights.double().cpu()
    gate_up, down, ids = gate_up.cpu(), down.cpu(), ids.long().cpu()
    out = torch.zeros(tokens, hidden, dtype=torch.float64)
    size, off = torch.zeros_like(out), torch.zeros_like(out)
    for t in range(tokens):
        if padding is not None and padding[t]:
            continue
        for k in range(ids.shape[1]):
            e = int(ids[t, k])
            if not 0 <= e < experts:
                continue
            w, g_rows, d = weights[t, k], gate_up[e].double(), down[e].double()
            both, both_size = g_rows @ x[t], g_rows.abs() @ x[t].abs()
            g, u = both[:width], both[width:]
            dg, du = chain(hidden) * both_size[:width], chain(hidden) * both_size[width:]
            p = phi(g, activation)
            a = w * p * u
            # |phi'| <= 1.13 for both activations; phi itself is evaluated in FP32:
            # the exponential's argument, of size |inner|, is off by 2 2^-23 |inner|,
            # and a dozen FP32 operations follow
            inner = g.abs() if activation == "silu" else 1.6 * (g.abs() + 0.045 * g.abs() ** 3)
            dp = 1.13 * dg + p.abs() * (2 * inner + 16) * STEP
            da = w.abs() * (dp * u.abs() + (p.abs() + dp) * du)
            out[t] += d @ a
            size[t] += d.abs() @ a.abs()
            # the activation as a sum of two BF16 numbers: half a step of half a step
            off[t] += d.abs() @ (da + HALF_BF16 ** 2 * (a.abs() + da))
    off = off + (chain(width) + ids.shape[1] * STEP) * (size + off)
    return out, off + HALF_BF16 * (out.abs() + off)


def routing(x: Tensor, router: Tensor, top_k: int, renormalise: bool = True,
            scale: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor]:
    """(ids, weights, relative bound of the FP32 weights) in float64."""
    x, router = x.double().cpu(), router.double().cpu()
    logits = x @ router.T
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids = order.indices[:, :top_k]
    kept = order.values[:, :top_k]
    base = kept if renormalise else logits
    weights = torch.exp(kept - torch.logsumexp(base, dim=-1, keepdim=True))
    # both logits of a quotient are off by chain(H) sum|x r|; exp of an FP32
    # argument d is off by (|d| + 2) 2^-23; the total adds at most 16 + 6 lane sums
    size = (x.abs() @ router.abs().T).amax(-1, keepdim=True)
    spread = (kept[:, :1] - kept).abs()
    bound = 2 * chain(x.shape[1]) * size + (2 * spread + 32) * STEP
    if scale is not None:
        weights = weights * scale.double().cpu()[ids]
    return ids, weights, bound


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantised(weights: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """(codes, scale bytes, float64 values) of weights [..., n], by the definition."""
    value = weights.double().cpu().unflatten(-1, (-1, 32))
    largest = value.abs().amax(-1)
    finite = torch.isfinite(largest)
    exponent = torch.frexp(torch.where(finite & (largest > 0), largest, 1.0)).exponent - 1
    exponent = torch.where(largest > 0, exponent, -1000)
    byte = torch.where(finite, (exponent + 125).clamp(2, 254), 255)
    scale = torch.ldexp(torch.ones_like(largest), byte - 127)
    quotient = (value / scale.unsqueeze(-1)).abs()
    grid = torch.tensor(E2M1, dtype=torch.float64)
    # nearest grid value; of two equally near the one with the even code
    # (codes count mantissa steps, so the last mantissa bit is the code's)
    distance = (quotient.unsqueeze(-1) - grid).abs() + torch.tensor([0, 1] * 4) * 1e-9
    distance = torch.where(torch.isfinite(distance), distance, 0.0)
    code = distance.argmin(-1)
    code = torch.where(finite.unsqueeze(-1), code, 0)
    negative = torch.signbit(value) & finite.unsqueeze(-1)
    values = torch.where(negative, -grid[code], grid[code]) * scale.unsqueeze(-1)
    values = torch.where(finite.unsqueeze(-1), values, math.nan).flatten(-2)
    nibble = (code + 8 * negative).flatten(-2)
    return (nibble[..., ::2] + 16 * nibble[..., 1::2]).to(torch.uint8), byte.to(torch.uint8), values


def values_of(codes: Tensor, scales: Tensor) -> Tensor:
    """float64 values of codes [..., n / 2] and scale bytes [..., n / 32]."""
    grid = torch.tensor([*E2M1, *(-v for v in E2M1)], dtype=torch.float64)
    codes, scales = codes.cpu().long(), scales.cpu().long()
    value = grid[torch.stack([codes % 16, codes // 16], -1).flatten(-2)]
    scale = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales - 127)
    scale = torch.where(scales == 255, math.nan, scale)
    return value * scale.repeat_interleave(32, -1)
