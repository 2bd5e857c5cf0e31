"""Ends of the norms' and joins' ranges (needs an MI355X): rows whose squares pass FP32,
epsilons of their size, and gradients summed over many rows."""

import pytest
import torch

from calibration_free_moe.reader.norms import join_block, norm_rows
from tests import block_reference as plain

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


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
