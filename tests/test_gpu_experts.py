"""routed_experts (cfmoe_routed_experts) against a float64 layer (needs an MI355X).

Outputs lie, element by element, within the bound that layer_reference derives
from the operands; masked and unrouted rows are exact zeros.
"""

import pytest
import torch

from calibration_free_moe.reader.experts import routed_experts
from calibration_free_moe.reader.microscale import Fp4Weights
from calibration_free_moe.reader.progressive import channel_major_down
from tests import layer_reference as plain

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


class Case:
    """A seeded layer and batch on the CPU, and its call on the GPU."""

    def __init__(self, tokens, hidden, width, experts, top_k, fp4=False, seed=0, zipf=False):
        g = torch.Generator().manual_seed(1000 * seed + tokens + width)
        self.fp4, self.experts = fp4, experts
        self.x = torch.randn(tokens, hidden, generator=g).bfloat16()
        self.x[:, ::90] *= 20
        shapes = {"gate_up": (experts, 2 * width, hidden), "down": (experts, hidden, width)}
        for name, shape in shapes.items():
            if fp4:
                codes = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), generator=g)
                scales = torch.randint(118, 124, (*shape[:-1], shape[-1] // 32), generator=g)
                setattr(self, name, Fp4Weights(codes.to(torch.uint8), scales.to(torch.uint8)))
            else:
                setattr(self, name, (torch.randn(shape, generator=g) * 0.02).bfloat16())
        score = torch.rand(tokens, experts, generator=g)
        if zipf:
            score = score ** (1 / torch.arange(1, experts + 1).float() ** -1.2)
        order = torch.sort(score, dim=-1, descending=True, stable=True).indices
        self.ids = order[:, :top_k].contiguous()
        self.weights = torch.softmax(torch.randn(tokens, top_k, generator=g), -1)
        self.padding = None

    def device_weights(self):
        if self.fp4:
            return tuple(Fp4Weights(w.codes.to(DEVICE), w.scales.to(DEVICE))
                         for w in (self.gate_up, self.down))
        return self.gate_up.to(DEVICE), channel_major_down(self.down.to(DEVICE))

    def values(self):
        if self.fp4:
            return tuple(plain.values_of(w.codes, w.scales) for w in (self.gate_up, self.down))
        return self.gate_up, self.down

    def run(self, activation="silu", out=None):
        gate_up, down = self.device_weights()
        padding = None if self.padding is None else self.padding.to(DEVICE)
        got = routed_experts(self.x.to(DEVICE), gate_up, down, self.ids.to(DEVICE),
                             self.weights.to(DEVICE), padding, out, activation=activation)
        torch.cuda.synchronize()
        return got

    def check(self, activation="silu"):
        got = self.run(activation).cpu().double()
        want, bound = plain.layer(self.x, *self.values(), self.ids, self.weights, self.padding,
                                  activation)
        worst = ((got - want).abs() / bound.clamp_min(1e-300)).max()
        assert bool(((got - want).abs() <= bound).all()), worst
        return got


SHAPES = [  # tokens, hidden, width, experts, top-k
    (1, 128, 32, 1, 1), (1, 2048, 768, 16, 8), (2, 256, 96, 4, 4), (3, 2816, 704, 8, 2),
    (5, 512, 160, 32, 6), (13, 384, 64, 3, 2), (16, 640, 352, 8, 3), (31, 256, 512, 64, 8),
    (40, 256, 64, 2, 1), (64, 256, 128, 8, 8), (100, 128, 96, 5, 3), (130, 256, 64, 2, 2),
    # about the largest batch that is not sorted
    (64, 256, 64, 70, 1), (65, 256, 64, 70, 1), (16, 256, 64, 20, 4), (13, 256, 64, 100, 5),
    # long rows and wide layers, few pairs an expert and many
    (3, 4096, 1056, 3, 2), (70, 4096, 64, 3, 2), (9, 1152, 2080, 2, 2), (60, 1152, 2080, 2, 2),
    (50, 2816, 96, 4, 2), (2, 128, 4096, 2, 1), (33, 128, 4096, 2, 2), (4, 128, 32, 4096, 64),
]


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_random_layers(shape, fp4):
    Case(*shape, fp4=fp4).check()


@pytest.mark.parametrize("width", [16, 48, 80, 272])
def test_widths_of_half_a_step(width):
    Case(9, 256, width, 6, 3).check()


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("weights_dtype", [torch.float32, torch.bfloat16])
def test_types_gelu_and_padding(fp4, ids_dtype, weights_dtype):
    for tokens in (4, 30):
        case = Case(tokens, 256, 96, 12, 3, fp4=fp4, seed=2)
        case.ids, case.weights = case.ids.to(ids_dtype), case.weights.to(weights_dtype)
        case.padding = torch.arange(tokens) % 4 == 1
        case.x[case.padding] = float("nan")  # what a padded row holds is never read
        got = case.check("gelu_tanh")
        assert bool((got[case.padding] == 0).all())


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
@pytest.mark.parametrize("tokens", [1, 3, 50])
def test_the_same_expert_twice_and_ids_of_no_expert(fp4, tokens):
    case = Case(tokens, 256, 64, 10, 4, fp4=fp4, seed=3)
    case.ids[:, 2] = case.ids[:, 0]
    case.ids[:, 3] = torch.tensor([-1, 10, 1 << 40])[torch.arange(tokens) % 3]
    case.check()
    case.ids[0] = -1
    got = case.check()
    assert bool((got[0] == 0).all())
    case.ids[:] = -5
    assert bool((case.run() == 0).all())
    case.ids[:] = 7
    case.check()


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
def test_every_row_padded(fp4):
    case = Case(6, 256, 64, 10, 4, fp4=fp4)
    case.padding = torch.ones(6, dtype=torch.bool)
    assert bool((case.run() == 0).all())


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
def test_skewed_routing_of_many_pairs(fp4):
    Case(300, 128, 64, 12, 4, fp4=fp4, zipf=True).check()


@pytest.mark.parametrize("shape", [
    (1750, 256, 256, 600, 4), (875, 128, 768, 300, 4), (1024, 128, 256, 300, 8),
    (1024, 128, 224, 300, 8), (800, 256, 512, 600, 4),
], ids=str)
@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
def test_rounds_of_several_tiles(shape, fp4):
    """So many runs that a workgroup has several tiles for each of its waves."""
    Case(*shape, fp4=fp4).check()


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
def test_the_largest_call(fp4):
    """8192 pairs; a sample of rows against the reference, more of them are refused."""
    case = Case(1024, 128, 32, 40, 8, fp4=fp4, seed=4)
    got = case.run().cpu().double()
    sample = torch.tensor([0, 1, 500, 777, 1023])
    want, bound = plain.layer(case.x[sample], *case.values(), case.ids[sample],
                              case.weights[sample])
    assert bool(((got[sample] - want).abs() <= bound).all())
    more = Case(1025, 128, 32, 40, 8, fp4=fp4)
    with pytest.raises(ValueError, match="8192"):
        more.run()


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
def test_infinities_reach_only_their_rows(fp4):
    """A NaN or infinity in a row of x, or in one expert's weights, leaves every
    row that does not use it as it was."""
    case = Case(20, 256, 64, 8, 2, fp4=fp4, seed=5)
    clean = case.run()
    case.x[7, 3] = float("inf")
    case.x[11, 200] = float("nan")
    if fp4:
        case.gate_up.scales[2, 5, 1] = 255
    else:
        case.gate_up[2, 5, 40] = float("nan")
        case.down[3, 9, 9] = float("inf")
    touched = (case.ids == 2).any(-1) | (case.ids == 3).any(-1)
    touched[7] = touched[11] = True
    assert 4 < int(touched.sum()) < 18
    got = case.run()
    assert torch.equal(got[~touched], clean[~touched])
    assert bool(got[11].isnan().all())
    assert bool(got[(case.ids == 2).any(-1)].isnan().all())


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
def test_repeats_are_bit_equal_and_out_is_written_whole(fp4):
    case = Case(50, 256, 96, 16, 4, fp4=fp4, seed=6)
    first = case.run()
    guard = torch.full((52, 256), 7.0, dtype=torch.bfloat16, device=DEVICE)
    for _ in range(3):
        out = guard[1:51]
        assert case.run(out=out) is out
        assert torch.equal(out, first)
        out.fill_(float("nan"))
    assert bool((guard[0] == 7).all()) and bool((guard[51] == 7).all())


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
def test_empty_batch(fp4):
    case = Case(1, 256, 64, 8, 2, fp4=fp4)
    gate_up, down = case.device_weights()
    got = routed_experts(case.x[:0].to(DEVICE), gate_up, down, case.ids[:0].to(DEVICE),
                         case.weights[:0].to(DEVICE))
    assert got.shape == (0, 256)


def test_offsets_past_32_bits():
    """Weights of more than 2^32 bytes: the last experts' rows are the ones read."""
    experts, hidden, width = 2200, 1024, 512
    gate_up = torch.zeros(experts, 2 * width, hidden, dtype=torch.bfloat16, device=DEVICE)
    down = torch.zeros(experts, width, hidden, dtype=torch.bfloat16, device=DEVICE).transpose(1, 2)
    assert gate_up.numel() * 2 > 1 << 32
    case = Case(2, hidden, width, 2, 2)
    gate_up[-2:], down[-2:] = case.gate_up.to(DEVICE), case.down.to(DEVICE)
    got = routed_experts(case.x.to(DEVICE), gate_up, down, (case.ids + experts - 2).to(DEVICE),
                         case.weights.to(DEVICE))
    want, bound = plain.layer(case.x, case.gate_up, case.down, case.ids, case.weights)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
@pytest.mark.parametrize("tokens", [2, 40])
def test_out_may_be_the_rows(tokens, fp4):
    case = Case(tokens, 256, 96, 16, 4, fp4=fp4, seed=8)
    want = case.run()
    rows = case.x.to(DEVICE)
    got = routed_experts(rows, *case.device_weights(), case.ids.to(DEVICE), case.weights.to(DEVICE),
                         None, rows)
    assert got is rows and torch.equal(rows, want)
