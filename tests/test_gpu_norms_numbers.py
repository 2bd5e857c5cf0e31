"""Ends of the norms' and joins' ranges (needs an MI355X): rows whose squares pass FP32,
and epsilons of their size."""

import pytest
import torch

from calibration_free_moe.reader.norms import norm_rows
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
