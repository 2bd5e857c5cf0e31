"""Plain 64-bit forms of what stands around a layer's experts (CPU), each with an
element-wise bound on what a right FP32 computation may be off.

With U = 2^-24, one FP32 rounding relative to its result:

* a sum of products goes through at most `chain` roundings, each of a partial sum no
  larger than the sum of magnitudes; a matrix instruction adds 32 products;
* a rounding to the outputs' type is off by half a step (`half_step`);
* an error of an operand passes on by the operation's derivative.
"""

from __future__ import annotations

import torch
from torch import Tensor

U = 2.0 ** -24


def half_step(dtype: torch.dtype) -> float:
    """Of one rounding to `dtype` after an FP32 computation, which an FP32 output is itself."""
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0


def within(got: Tensor, want: Tensor, bound: Tensor) -> None:
    """`bound` is that of the FP32 value; got's own rounding comes on top."""
    half = half_step(got.dtype)
    error = (got.detach().cpu().double() - want).abs()
    allowed = bound + half * (want.abs() + bound) + 1e-44
    worst = (error / allowed).max() if error.numel() else 0.0
    assert got.shape == want.shape and bool((error <= allowed).all()), float(worst)


# ---------------------------------------------------------------------------
# rows by expert


def order(ids: Tensor, experts: int, padding: Tensor | None) -> tuple[list, list, list]:
    """(offsets, places, pairs) one pair after the other."""
    lists = [[] for _ in range(experts + 1)]
    for t, row in enumerate(ids.tolist()):
        for k, e in enumerate(row):
            kept = 0 <= e < experts and not (padding is not None and padding[t])
            lists[e if kept else experts].append(t * len(row) + k)
    offsets, pairs, places = [0], [], [0] * ids.numel()
    for e, members in enumerate(lists):
        for pair in members:
            places[pair] = len(pairs) if e < experts else -1 - len(pairs)
            pairs.append(pair)
        offsets.append(len(pairs))
    return offsets[:-1], places, pairs


def gather(hidden: Tensor, places: Tensor) -> Tensor:
    tokens, top_k = places.shape
    rows = torch.zeros(tokens * top_k, hidden.shape[1], dtype=hidden.dtype)
    t, k = torch.nonzero(places >= 0, as_tuple=True)
    rows[places[t, k].long()] = hidden[t]
    return rows


def combine(rows: Tensor, places: Tensor, weights: Tensor | None) -> tuple[Tensor, Tensor]:
    """(out, bound): a product and an addition a slot."""
    rows = rows.double()
    out = torch.zeros(places.shape[0], rows.shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    for k in range(places.shape[1]):
        t = torch.nonzero(places[:, k] >= 0).flatten()
        row = rows[places[t, k].long()]
        if weights is not None:
            row = row * weights[t, k].double().unsqueeze(-1)
        out[t] += row
        size[t] += row.abs()
    return out, places.shape[1] * U * size


def combine_backward(grad: Tensor, rows: Tensor, places: Tensor, weights: Tensor | None):
    """(drows, its bound, dweights, its bound)."""
    grad, rows = grad.double(), rows.double()
    hidden = rows.shape[1]
    drows, dweights = torch.zeros_like(rows), torch.zeros(places.shape, dtype=torch.float64)
    size = torch.zeros_like(dweights)
    t, k = torch.nonzero(places >= 0, as_tuple=True)
    row = places[t, k].long()
    w = 1.0 if weights is None else weights[t, k].double().unsqueeze(-1)
    drows[row] = grad[t] * w
    dweights[t, k] = (grad[t] * rows[row]).sum(-1)
    size[t, k] = (grad[t] * rows[row]).abs().sum(-1)
    # a lane adds hidden / 256 and up to 8 products, then 6 lane steps and 4 waves
    return drows, U * drows.abs(), dweights, (hidden / 256 + 8 + 6 + 4) * U * size


# ---------------------------------------------------------------------------
# norms and joins

# A row's sum: 8 values of a thread, 6 lane steps, 16 waves; then a division, epsilon,
# a root (halving what is relative) and a reciprocal.
ROW = 8 + 6 + 16
ROOT = (ROW + 2) / 2 + 2


def unit(v: Tensor, epsilon: float) -> tuple[Tensor, Tensor]:
    inverse = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + epsilon)
    return v * inverse, inverse


def join(hidden, block, post, gate, scale, following, epsilon):
    """(joined, next) in 64 bits; differentiable."""
    joined = hidden
    if block is not None:
        n = block if post is None else unit(block, epsilon)[0] * post
        joined = scale * hidden + (n if gate is None else gate * n)
    out = None if following is None else unit(joined, epsilon)[0] * following
    return joined, out


def join_bounds(hidden, block, post, gate, scale, following, epsilon, grad_joined=None,
                grad_out=None) -> dict:
    """Bounds of joined and next and of each gradient, from the operands (64 bits)."""
    bounds, tokens = {}, hidden.shape[0]
    g = torch.ones_like(hidden) if gate is None else gate.expand_as(hidden)
    size = hidden.shape[1]
    if block is None:
        joined, e_joined = hidden, torch.zeros_like(hidden)
    else:
        p = torch.ones_like(hidden) if post is None else post.expand_as(hidden)
        b, inverse_b = (block, 1.0) if post is None else unit(block, epsilon)
        e_b = 0 * b if post is None else (ROOT + 1) * U * b.abs()
        n = b * p
        e_n = e_b * p.abs() + U * n.abs()
        joined = scale * hidden + g * n
        # the scale is an FP32 number; one rounding of the gate's product, one of the sum
        e_joined = g.abs() * e_n + U * ((scale * hidden).abs() + (g * n).abs() + joined.abs())
        bounds["joined"] = e_joined
    if following is not None:
        j, inverse = unit(joined, epsilon)
        # the mean's own error, from those of its terms
        drift = ((joined.abs() * e_joined).sum(-1, keepdim=True)
                 / (joined * joined).sum(-1, keepdim=True).clamp_min(1e-300))
        e_j = inverse * e_joined + j.abs() * (drift + (ROOT + 1) * U)
        bounds["out"] = e_j * following.abs() + U * (j * following).abs()
    if grad_joined is None and grad_out is None:
        return bounds
    grad = torch.zeros_like(hidden) if grad_joined is None else grad_joined
    e_grad = torch.zeros_like(hidden)
    # a workgroup's rows, then its fellows' sums and the waves' (tokens of at least one group)
    chain = tokens / 1024 + 1 + 64 + 16 + 1

    def over_rows(value, error):
        return error.sum(0) + chain * U * value.abs().sum(0)

    def back(grad, e_grad, u, e_u, inverse, drift):
        """Of inverse (grad - u mean(grad u))."""
        mean = (grad * u).mean(-1, keepdim=True)
        e_mean = ((e_grad * u.abs() + grad.abs() * e_u).mean(-1, keepdim=True)
                  + (ROW + 3) * U * (grad * u).abs().mean(-1, keepdim=True))
        inner = grad.abs() + (u * mean).abs()
        return inverse * (e_grad + e_u * mean.abs() + u.abs() * e_mean
                          + (drift + (ROOT + 3) * U) * inner), inverse * (grad - u * mean)

    if grad_out is not None:
        bounds["next"] = over_rows(grad_out * j, grad_out.abs() * e_j)
        y = grad_out * following
        e_y, value = back(y, U * y.abs(), j, e_j, inverse, drift)
        grad = grad + value
        e_grad = e_y + U * grad.abs()
    bounds["hidden"] = abs(scale) * e_grad + 2 * U * (scale * grad).abs()
    if block is None:
        return bounds
    both, e_both = grad * n, e_grad * n.abs() + grad.abs() * e_n + U * (grad * n).abs()
    if gate is not None:
        if gate.dim() == 1:
            bounds["gate"] = over_rows(both, e_both)
        elif gate.shape[1] == 1 and size > 1:
            bounds["gate"] = e_both.sum(-1, keepdim=True) + ROW * U * both.abs().sum(-1, keepdim=True)
        else:
            bounds["gate"] = e_both
    dn, e_dn = grad * g, e_grad * g.abs() + U * (grad * g).abs()
    if post is None:
        bounds["block"] = e_dn
    else:
        bounds["post"] = over_rows(dn * b, e_dn * b.abs() + dn.abs() * e_b)
        inner = dn * p
        bounds["block"] = back(inner, e_dn * p.abs() + U * inner.abs(), b, e_b, inverse_b, 0.0)[0]
    return bounds


# ---------------------------------------------------------------------------
# adapters


def adapters(base, hidden, encoder, decoder, slots, scales) -> tuple[Tensor, Tensor]:
    """(out, bound): the inner values are held to 2^-16."""
    out, x = base.double(), hidden.double()
    bound = torch.zeros_like(out)

    def chain(products):
        # 32 products inside an instruction, the instructions, 16 waves and the ends
        return (32 + products / 32 + 16 + 4) * 2 * U

    for t, a in enumerate(slots.tolist()):
        if not 0 <= a < encoder.shape[0]:
            continue
        c, d = encoder[a].double(), decoder[a].double()
        s = 1.0 if scales is None else float(scales[a])
        v = s * (c @ x[t])
        e_v = abs(s) * chain(x.shape[1]) * (c.abs() @ x[t].abs()) + 2 * U * v.abs()
        e_v = e_v + 2.0 ** -16 * (v.abs() + e_v)
        out[t] += d @ v
        bound[t] = d.abs() @ e_v + 2 * chain(2 * c.shape[0]) * (d.abs() @ v.abs()) + U * out[t].abs()
    return out, bound
