"""route and routed_experts at the ends of their operands' ranges: logits beyond FP32,
infinite weights, activations next to the largest number, a layer of one expert (needs
an MI355X).
"""

import pytest
import torch

from calibration_free_moe.reader.experts import routed_experts
from calibration_free_moe.reader.progressive import channel_major_down
from calibration_free_moe.reader.router import route
from tests import layer_reference as plain
from tests.test_gpu_experts import Case

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


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
@pytest.mark.parametrize("tokens,experts", [(1, 8), (3, 8), (20, 16), (60, 4)])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -118], ids=["", "small"])
def test_infinite_down_weights(tokens, experts, fp4, scale):
    """An infinite weight of `down` makes its output infinite, of the products' sign, NaN
    where two of them disagree, and leaves the outputs beside it as they are."""
    case = Case(tokens, 256, 96, experts, 2, fp4=fp4, seed=11)
    case.weights = case.weights * scale
    g = torch.Generator().manual_seed(12)
    for e in range(experts):
        for h in torch.randperm(256, generator=g)[:40].tolist():
            channel = int(torch.randint(96, (1,), generator=g))
            negative = int(torch.randint(2, (1,), generator=g))
            if fp4:  # 6 2^127, beyond BF16, alone in its block
                case.down.codes[e, h, channel // 32 * 16:channel // 32 * 16 + 16] = 0
                case.down.codes[e, h, channel // 2] = (7 + 8 * negative) << 4 * (channel % 2)
                case.down.scales[e, h, channel // 32] = 254
            else:
                case.down[e, h, channel] = -float("inf") if negative else float("inf")
    gate_up, down = case.values()
    if fp4:
        down = down.float().bfloat16()
    want, bound = plain.layer(case.x, gate_up, down, case.ids, case.weights)
    assert 20 * tokens < int(want.isinf().sum()) and int(want.isnan().sum()) < 20 * tokens
    got = case.run().cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    finite = want.isfinite()
    # (2^-132: what the smallest activations' second part may be off, times 96 weights
    # below 2^7)
    assert bool(((got - want).abs() <= bound + 96 * 2.0 ** -125)[finite].all())


@pytest.mark.parametrize("weight", [3.4e38, -3.4e38, 3.2e38])
def test_activations_next_to_the_largest_number(weight):
    """3.4e38 lies beyond half a step of the largest BF16 number and is an FP32 one."""
    x = torch.zeros(1, 128, dtype=torch.bfloat16)
    gate_up = torch.zeros(1, 64, 128, dtype=torch.bfloat16)
    down = torch.zeros(1, 128, 32, dtype=torch.bfloat16)
    x[0, 0], gate_up[0, 0, 0], gate_up[0, 32, 0] = 1, 32, 2.0 ** -5  # silu(32) / 32 = 1 in FP32
    down[0, :, 0] = 2.0 ** -20
    got = routed_experts(x.to(DEVICE), gate_up.to(DEVICE), channel_major_down(down.to(DEVICE)),
                         torch.zeros(1, 1, dtype=torch.int32, device=DEVICE),
                         torch.tensor([[weight]], device=DEVICE))
    want = torch.tensor(weight).double() * 2.0 ** -20
    # an FP32 exponential and quotient, 2^-16 of the activation, one rounding
    off = 16 * plain.STEP + plain.HALF_BF16 ** 2 + plain.HALF_BF16
    assert bool(((got.cpu().double() - want).abs() <= 1.01 * off * want.abs()).all())


def test_a_layer_of_one_expert_as_a_view():
    """The stride of a dimension of size one says nothing: a shared expert's channel-major
    down [H, I] with a leading dimension is a layer's."""
    case = Case(5, 256, 96, 1, 1, seed=13)
    gate_up, down = case.device_weights()
    one = down[0][None]
    assert one.stride() == (256, 1, 256) and channel_major_down(one).stride() == one.stride()
    rest = (case.ids.to(DEVICE), case.weights.to(DEVICE))
    got = routed_experts(case.x.to(DEVICE), gate_up[0][None], one, *rest)
    assert torch.equal(got, routed_experts(case.x.to(DEVICE), gate_up, down, *rest))


@pytest.mark.parametrize("renormalise", [True, False])
def test_logits_beyond_fp32_among_many_tokens(renormalise):
    """The kernel of many tokens: the rows that overflow, and the ordinary ones beside them."""
    g = torch.Generator().manual_seed(14)
    x = torch.randn(1400, 256, generator=g).bfloat16()
    router = (torch.randn(200, 256, generator=g) * 0.1).bfloat16()
    large = torch.arange(1400) % 9 == 4
    x[large] = torch.where(x[large] < 0, -3e38, 3e38).bfloat16()
    ids, weights = route(x.to(DEVICE), router.to(DEVICE), 5, renormalise=renormalise)
    want_ids, want, bound = plain.routing(x, router, 5, renormalise)
    assert torch.equal(ids.cpu().long(), want_ids)
    # (differences of 1e36 and more: the first expert has all the weight)
    assert bool((want[large, 0] == 1).all()) and torch.equal(weights.cpu()[large].double(), want[large])
    rest = ~large
    assert bool(((weights.cpu().double() - want).abs() <= bound * want)[rest].all())
