"""route and routed_experts at the ends of their operands' ranges: logits beyond FP32,
infinite weights, activations next to the largest number, a layer of one expert (needs
an MI355X).
"""

import pytest
import torch

from calibration_free_moe.reader.router import route
from tests import layer_reference as plain

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


@pytest.mark.parametrize("experts,top_k", [(1, 1), (5, 4), (5, 5), (20, 6), (64, 63), (200, 7)])
@pytest.mark.parametrize("renormalise", [True, False])
def test_weights_of_logits_beyond_fp32(experts, top_k, renormalise):
    """Row 1's largest products cancel exactly, row 2's logits are all beyond FP32.

    FP64 dot products settle both rows, so a weight is off by the FP32 exponential of
    a difference d, (|d| + 2) 2^-23, and a total of at most 16 + 6 additions.
    """
    hidden = 512
    g = torch.Generator().manual_seed(experts + top_k)
    x = torch.randn(4, hidden, generator=g).bfloat16()
    router = (torch.randn(experts, hidden, generator=g) * 0.1).bfloat16()
    x[:, 8:10] = 0
    x[1, 8:10] = 3e38
    router[:, 8] = torch.randint(2, 8, (experts,), generator=g).bfloat16()
    router[:, 9] = -router[:, 8]
    x[2] = torch.where(x[2] < 0, -3e38, 3e38).bfloat16()
    ids, weights = route(x.to(DEVICE), router.to(DEVICE), top_k, renormalise=renormalise)
    plain_x = x.clone()
    plain_x[1, 8:10] = 0
    want_ids, want, bound = plain.routing(plain_x, router, top_k, renormalise)
    logits = plain_x.double() @ router.double().T
    kept = logits.gather(1, want_ids)
    exact = (2 * (kept[:, :1] - kept) + 32) * plain.STEP
    bound[1:3] = exact[1:3]
    assert torch.equal(ids.cpu().long(), want_ids)
    assert bool(((weights.cpu().double() - want).abs() <= bound * want + 2.0 ** -126).all())
