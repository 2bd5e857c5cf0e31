"""routed_experts through every kernel that its rules can choose, against a float64 layer
(needs an MI355X). tests/test_layer_dispatch.py asserts that the cases leave none out.
"""

import pytest
import torch

from calibration_free_moe.reader.experts import routed_experts
from calibration_free_moe.reader.microscale import Fp4Weights
from tests import layer_reference as plain
from tests.layer_dispatch import CASES

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


def padded(rows, experts):
    """The few experts' rows on the GPU, zeros for the others."""
    to = torch.zeros((experts, *rows.shape[1:]), dtype=rows.dtype, device=DEVICE)
    to[: rows.shape[0]] = rows.to(DEVICE)
    return to


@pytest.mark.parametrize("hidden,width,experts,pairs,fp4,counts", CASES,
                         ids=["-".join(map(str, case[:4])) + ("-fp4" if case[4] else "") for case in CASES])
def test_every_kernel(hidden, width, experts, pairs, fp4, counts):
    g = torch.Generator().manual_seed(hidden + width + pairs)
    ids = torch.full((pairs,), -1)
    ids[: sum(counts)] = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    ids = ids[torch.randperm(pairs, generator=g)].unsqueeze(1)
    weights = torch.rand(pairs, 1, generator=g) + 0.5
    x = torch.randn(pairs, hidden, generator=g).bfloat16()
    x[:, ::90] *= 20
    values, given = [], []
    for rows, length in ((2 * width, hidden), (hidden, width)):
        if fp4:
            codes = torch.randint(0, 256, (len(counts), rows, length // 2), generator=g).to(torch.uint8)
            scales = torch.randint(118, 124, (len(counts), rows, length // 32), generator=g).to(torch.uint8)
            values.append(plain.values_of(codes, scales))
            given.append(Fp4Weights(padded(codes, experts), padded(scales, experts)))
        else:
            values.append((torch.randn(len(counts), rows, length, generator=g) * 0.02).bfloat16())
            given.append(values[-1])
    if not fp4:
        given = [padded(given[0], experts), padded(given[1].transpose(1, 2), experts).transpose(1, 2)]
    got = routed_experts(x.to(DEVICE), *given, ids.to(DEVICE), weights.to(DEVICE)).cpu().double()
    want, bound = plain.layer(x, *values, ids, weights)
    assert bool(((got - want).abs() <= bound).all()), ((got - want).abs() / bound.clamp_min(1e-300)).max()
