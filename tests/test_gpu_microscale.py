"""quantise_fp4 and dequantise_fp4 against the definition in float64 (needs an MI355X).

Codes, scale bytes and values are integers or exact: every comparison is for
equality.
"""

import pytest
import torch

from calibration_free_moe.reader.microscale import Fp4Weights, dequantise_fp4, quantise_fp4
from tests import layer_reference as plain

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


def check(weights):
    got = quantise_fp4(weights.to(DEVICE))
    values = dequantise_fp4(got)
    torch.cuda.synchronize()
    codes, scales, want = plain.quantised(weights)
    assert got.shape == weights.shape and got.codes.shape == codes.shape
    assert torch.equal(got.scales.cpu(), scales)
    assert torch.equal(got.codes.cpu(), codes)
    values = values.cpu()
    assert values.dtype == torch.bfloat16
    assert torch.equal(values.double().nan_to_num(nan=1e300), want.nan_to_num(nan=1e300))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(32,), (1, 32), (3, 96), (2, 5, 64), (7, 2816), (257, 160)])
def test_random_weights(dtype, shape):
    g = torch.Generator().manual_seed(sum(shape))
    check((torch.randn(shape, generator=g) * 0.02).to(dtype))


def test_every_bf16_value_beside_a_larger_one():
    """All finite BF16 values, each block's scale set by a value of its first place."""
    bits = torch.arange(1 << 16, dtype=torch.int32)
    value = (bits << 16).view(torch.float32).bfloat16()
    value = value[value.isfinite()]
    order = value.float().abs().argsort(stable=True)
    value = value[order]
    value = value[: value.numel() // 31 * 31].reshape(-1, 31)
    for lead in (1.0, 6.0, 2.0 ** -120, 3.0e38):
        block = torch.cat([torch.full((value.shape[0], 1), lead).bfloat16(), value], 1)
        check(block)
    check(torch.cat([value[:, :1], value], 1))


def test_ties_and_borders():
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9])
    near = torch.cat([border, torch.nextafter(border, torch.tensor(0.0)),
                      torch.nextafter(border, torch.tensor(9.0))])
    block = torch.cat([torch.tensor([4.0]), near, torch.tensor([-0.0])])
    for power in (-127, -126, -120, -30, -3, 0, 5, 100, 125):
        scaled = (block.double() * 2.0 ** power).float()
        check(torch.stack([scaled, -scaled]))


def test_blocks_that_hold_no_scale():
    block = torch.zeros(6, 64)
    block[1, 3] = float("nan")
    block[2, 40] = float("inf")
    block[3, 41] = -float("inf")
    block[4, 5] = -0.0
    block[5, 6] = 2.0 ** -149
    for dtype in (torch.float32, torch.bfloat16):
        check(block.to(dtype))


def test_values_of_every_code_and_scale():
    scales = torch.arange(256, dtype=torch.uint8).reshape(256, 1)
    codes = torch.arange(16, dtype=torch.uint8).repeat(256, 1) * 17
    got = dequantise_fp4(Fp4Weights(codes.to(DEVICE), scales.to(DEVICE))).cpu()
    want = plain.values_of(codes, scales)
    # (6 2^127 is the one magnitude beyond BF16: scale byte 254, codes above 3)
    want = want.float().bfloat16().double()
    assert torch.equal(got.double().nan_to_num(nan=1e300, posinf=2e300, neginf=-2e300),
                       want.nan_to_num(nan=1e300, posinf=2e300, neginf=-2e300))


def test_empty_weights():
    got = quantise_fp4(torch.empty(0, 64, dtype=torch.bfloat16, device=DEVICE))
    assert got.shape == (0, 64) and dequantise_fp4(got).shape == (0, 64)


def test_more_lanes_than_a_launch_holds():
    """A grid that walks: over 2^28 lanes of eight values, checked in its parts."""
    rows = 270_000
    weights = torch.empty(rows, 8192, dtype=torch.bfloat16, device=DEVICE)
    g = torch.Generator(device=DEVICE).manual_seed(1)
    weights.normal_(0.0, 0.02, generator=g)
    got = quantise_fp4(weights)
    values = dequantise_fp4(got)
    for begin in (0, 131_000, 262_140, rows - 5):
        part = slice(begin, begin + 5)
        codes, scales, want = plain.quantised(weights[part])
        assert torch.equal(got.codes[part].cpu(), codes)
        assert torch.equal(got.scales[part].cpu(), scales)
        assert torch.equal(values[part].cpu().double(), want)
