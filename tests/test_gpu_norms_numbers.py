"""Ends of the norms' and joins' ranges (needs an MI355X): rows whose squares pass FP32
in either norm or both, epsilons of their size, and gradients summed over many rows."""

import pytest
import torch

from calibration_free_moe.reader.norms import join_block, norm_rows
from tests import block_reference as plain

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("size", [40, 500, 2048, 8192])
@pytest.mark.parametrize("epsilon", [1e30, 1e25, 1e-6])
def test_epsilon_beside_rows_whose_squares_pass_fp32(size, epsilon):
    """Rows of one magnitude from below the largest sum of squares to far above it."""
    edge = (3.4e38 / size) ** 0.5
    rows = torch.tensor([0.5, 0.99, 1.001, 1.1, 3.0, 100.0]).unsqueeze(-1) * edge
    signs = 1 - 2.0 * (torch.arange(size) % 3 % 2)
    x = (rows * signs).float()
    w = 1 + torch.randn(size, generator=torch.Generator().manual_seed(1)) / 10
    on, weight = x.to(DEVICE).requires_grad_(), w.to(DEVICE).requires_grad_()
    exact, exact_w = x.double().requires_grad_(), w.double().requires_grad_()
    out = norm_rows(on, weight, epsilon=epsilon)
    want = plain.join(exact, None, None, None, 1.0, exact_w, epsilon)[1]
    grad = torch.randn(x.shape, generator=torch.Generator().manual_seed(2))
    bounds = plain.join_bounds(x.double(), None, None, None, 1.0, w.double(), epsilon, None,
                               grad.double())
    # epsilon is an FP32 number and so is its scaled one: two roundings more, halved by the root
    plain.within(out, want.detach(), bounds["out"] + plain.U * want.detach().abs())
    got = torch.autograd.grad(out, (on, weight), grad.to(DEVICE))
    wanted = torch.autograd.grad(want, (exact, exact_w), grad.double())
    # (the same in the gradients, where the root stands three times; below 2^-126 a step is
    # 2^-149)
    _, inverse = plain.unit(x.double(), epsilon)
    terms = inverse * (grad.double() * w.double()).abs().max(-1, keepdim=True).values
    plain.within(got[0], wanted[0], bounds["hidden"] + 4 * plain.U * terms + 2.0 ** -148)
    plain.within(got[1], wanted[1], bounds["next"] + 2 * plain.U * grad.double().abs().sum(0))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("size", [5, 40, 264, 1001, 4096, 8192])
@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
def test_joins_of_rows_whose_squares_pass_fp32(dtype, size, gate):
    """The norm behind the block, the one of the join, and both, beside ordinary rows."""
    g = torch.Generator().manual_seed(size)

    def numbers(*shape):
        return torch.randn(shape, generator=g).clamp(-2.5, 2.5)

    block = numbers(7, size) * torch.tensor([1, 1e21, 1e30, 1, 1e25, 3e37, 1e-20]).unsqueeze(-1)
    hidden = numbers(7, size) * torch.tensor([1, 1, 1e-3, 1e30, 1e22, 3e37, 1]).unsqueeze(-1)
    shape = {"none": None, "channel": (size,), "row": (7, 1), "full": (7, size)}[gate]
    made = {"hidden": hidden.to(dtype), "block": block.to(dtype),
            "post": (1 + numbers(size) / 10).to(dtype),
            "gate": None if shape is None else (1 + numbers(*shape) / 10).to(dtype),
            "next": (1 + numbers(size) / 10).to(dtype)}
    scale = 0.75
    on = {k: None if v is None else v.to(DEVICE).requires_grad_() for k, v in made.items()}
    exact = {k: None if v is None else v.double().requires_grad_() for k, v in made.items()}
    outputs = join_block(on["hidden"], on["block"], post_weight=on["post"], gate=on["gate"],
                         residual_scale=scale, next_weight=on["next"])
    want = plain.join(exact["hidden"], exact["block"], exact["post"], exact["gate"], scale,
                      exact["next"], 1e-6)
    grads = [numbers(7, size).to(dtype) for _ in range(2)]
    operands = [None if exact[k] is None else exact[k].detach() for k in ("hidden", "block", "post", "gate")]
    bounds = plain.join_bounds(*operands, scale, exact["next"].detach(), 1e-6,
                               *(v.double() for v in grads))
    # the steps of scaled rows are by powers of two, exact but below 2^-126 (a step of 2^-149
    # in FP32, of 2^-133 in BF16, against values of 1); a root of the scaled sum is one more
    step = 2.0 ** -133 if dtype == BF16 else 2.0 ** -148
    for got, right, name in zip(outputs, want, ("joined", "out")):
        plain.within(got, right.detach(), bounds[name] + plain.U * right.detach().abs() + step)
    names = [k for k, v in on.items() if v is not None]
    got = torch.autograd.grad(outputs, [on[k] for k in names], [v.to(DEVICE) for v in grads])
    wanted = torch.autograd.grad(want, [exact[k] for k in names], [v.double() for v in grads])
    for name, a, b in zip(names, got, wanted):
        assert bool(a.isfinite().all()), name
        plain.within(a, b, bounds[name] * 1.01 + 2 * plain.U * b.abs() + step)
    # a row's results are its own: the same bits without the others
    for t in range(7):
        alone = [v[t:t + 1] if v is not None and v.dim() == 2 else v
                 for v in (on[k] for k in ("hidden", "block", "post", "gate", "next"))]
        again = join_block(alone[0], alone[1], post_weight=alone[2], gate=alone[3],
                           residual_scale=scale, next_weight=alone[4])
        assert torch.equal(again[0][0], outputs[0][t]) and torch.equal(again[1][0], outputs[1][t])


@pytest.mark.parametrize("tokens,size", [(515, 1003), (1024, 64), (1024, 700)])
@pytest.mark.parametrize("large", [0, 16, 400])
def test_gradients_summed_over_rows_pass_few_roundings(tokens, size, large):
    """A row of 1 among rows of 2^-25, each of which an FP32 sum of 1 loses. Every row has a
    workgroup of its own here; of their sums 16 waves take every 16th, in 8 sums each, and
    both are added in pairs: tokens / 128 roundings, 3 and 4."""
    rows = torch.full((tokens, size), 2.0 ** -25)
    rows[large] = 1
    want = torch.full((size,), 1 + (tokens - 1) * 2.0 ** -25, dtype=torch.float64)
    allowed = ((tokens + 127) // 128 + 3 + 4) * plain.U * want
    grad, ones = rows.to(DEVICE), torch.ones(tokens, size, device=DEVICE)
    # (rows of ones have the root 1, so that each gradient is the sum of `rows`)
    for which in ("next", "post", "gate"):
        w = torch.ones(size, device=DEVICE, requires_grad=True)
        if which == "next":
            out = norm_rows(ones, w, epsilon=1e-30)
        elif which == "post":
            out = join_block(0 * ones, ones, post_weight=w, epsilon=1e-30)
        else:
            out = join_block(0 * ones, ones, gate=w)
        (got,) = torch.autograd.grad(out, w, grad)
        plain.within(got, want, allowed)
