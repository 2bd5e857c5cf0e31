"""route (cfmoe_route) against a float64 router (needs an MI355X).

Ids must equal those of the exact logits everywhere, near ties and ties among
them; weights lie within the bound that layer_reference derives, plus half a BF16
step where they are BF16.
"""

import pytest
import torch

from calibration_free_moe.reader.router import route
from tests import layer_reference as plain

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


def rows(tokens, hidden, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens, hidden, generator=g) * std).bfloat16()


def check(x, router, top_k, **options):
    ids, weights = route(x.to(DEVICE), router.to(DEVICE), top_k, **options)
    torch.cuda.synchronize()
    scale = options.get("expert_scale")
    want_ids, want, bound = plain.routing(x, router, top_k, options.get("renormalise", True), scale)
    assert ids.dtype == options.get("ids_dtype", torch.int32)
    assert weights.dtype == options.get("weights_dtype", torch.float32)
    assert torch.equal(ids.cpu().long(), want_ids)
    if weights.dtype == torch.bfloat16:
        bound = bound + plain.HALF_BF16 * (1 + bound)
    error = (weights.cpu().double() - want).abs()
    assert bool((error <= bound * want.abs() + 2.0 ** -126).all()), (error / want).max()


@pytest.mark.parametrize("tokens,hidden,experts,top_k", [
    (1, 128, 1, 1), (1, 2048, 128, 8), (2, 256, 8, 8), (15, 384, 17, 3), (16, 640, 64, 6),
    (17, 2816, 128, 8), (33, 1024, 65, 1), (130, 2048, 256, 8), (300, 512, 250, 10),
    (5, 256, 1024, 64), (3, 256, 64, 64), (4, 4096, 513, 33), (2, 65536, 20, 4),
    (300, 2176, 1000, 3), (900, 4480, 300, 5),
])
@pytest.mark.parametrize("renormalise", [True, False])
def test_random_rows(tokens, hidden, experts, top_k, renormalise):
    x = rows(tokens, hidden, tokens + hidden)
    x[:, :: 100] *= 20
    router = rows(experts, hidden, experts + 7, 0.02)
    check(x, router, top_k, renormalise=renormalise)


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("weights_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scaled", [False, True])
def test_types_and_scale(ids_dtype, weights_dtype, scaled):
    x, router = rows(21, 256, 3), rows(40, 256, 4, 0.1)
    scale = (torch.rand(40, generator=torch.Generator().manual_seed(5)) + 0.5).to(DEVICE)
    check(x, router, 5, ids_dtype=ids_dtype, weights_dtype=weights_dtype,
          expert_scale=scale if scaled else None)


def test_order_of_the_exact_logits():
    """Experts whose logits differ by less than an FP32 sum is off: pairs of rows
    that differ in one coordinate where x is tiny, the larger at either place."""
    hidden, experts = 2048, 32
    x = rows(64, hidden, 11)
    router = rows(experts, hidden, 12, 0.5)
    x[:, 77] = 2.0 ** -24
    for e in range(0, experts, 2):
        router[e, 77], router[e + 1, 77] = (1.0, 1.5) if e % 4 else (1.5, 1.0)
        router[e + 1, :77], router[e + 1, 78:] = router[e, :77], router[e, 78:]
    logits = x.double() @ router.double().T
    gap = (logits[:, ::2] - logits[:, 1::2]).abs()
    assert bool(((gap - 2.0 ** -25).abs() < 2.0 ** -40).all())
    check(x, router, 9)


def test_ties_go_to_the_lowest_expert():
    x, router = rows(9, 256, 13), rows(20, 256, 14, 0.1)
    router[5] = router[2]
    router[17] = router[2]
    router[11] = router[10]
    check(x, router, 20)
    check(x, torch.zeros(20, 256, dtype=torch.bfloat16), 6)
    check(torch.zeros(3, 256, dtype=torch.bfloat16), -router, 6)


def test_rows_that_are_not_finite():
    """NaN ranks above all (as torch.topk), ids stay distinct and inside [0, E)."""
    x, router = rows(6, 256, 15), rows(70, 256, 16, 0.1)
    x[1, 3] = float("nan")
    x[2, 9] = float("inf")
    x[3] = 3e38
    router[44, 5] = float("nan")
    ids, weights = route(x.to(DEVICE), router.to(DEVICE), 7)
    ids, weights = ids.cpu(), weights.cpu()
    for row in ids.tolist():
        assert len(set(row)) == 7 and all(0 <= e < 70 for e in row)
    assert ids[1].tolist() == [0, 1, 2, 3, 4, 5, 6] and bool(weights[1].isnan().all())
    assert ids[0, 0] == 44 and ids[4, 0] == 44
    others = torch.arange(70) != 44
    want = (x[0].double() @ router[others].double().T).argsort(descending=True)[:6]
    want = torch.where(want >= 44, want + 1, want)
    assert ids[0, 1:].tolist() == want.tolist()
    # logits beyond FP32's range keep their order
    exact = x[3].double() @ router[others].double().T
    want = exact.argsort(descending=True, stable=True)[:6]
    assert ids[3, 1:].tolist() == torch.where(want >= 44, want + 1, want).tolist()


def test_out_and_empty_batches():
    x, router = rows(5, 128, 17).to(DEVICE), rows(12, 128, 18).to(DEVICE)
    ids, weights = route(x, router, 4, ids_dtype=torch.int64)
    out = (torch.full_like(ids, -1), torch.full_like(weights, -1.0))
    got = route(x, router, 4, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    assert torch.equal(out[0], ids) and torch.equal(out[1], weights)
    ids, weights = route(x[:0], router, 4)
    assert ids.shape == weights.shape == (0, 4)


@pytest.mark.parametrize("hidden,experts", [(512, 256), (128, 100), (2816, 130), (4096, 128)])
def test_many_tokens(hidden, experts):
    """The kernel of many tokens (over 1024 tiles of 16 experts and 16 tokens)."""
    tokens = 16 * (1024 // ((experts + 15) // 16)) + 21
    x, router = rows(tokens, hidden, 19), rows(experts, hidden, 20, 0.02)
    x[:, :: 100] *= 20
    router[7] = router[3]
    check(x, router, 8)
    check(x, router, 3, renormalise=False, ids_dtype=torch.int64)


def test_open_order_about_the_cut():
    """More experts than are kept lie within an FP32 sum's error of the cut."""
    hidden, experts = 1024, 48
    x, router = rows(40, hidden, 21), rows(experts, hidden, 22, 0.5)
    x[:, 5] = 2.0 ** -26
    for e in range(8, 40):
        router[e] = router[8]
        router[e, 5] = 1.0 + (e * 11 % 32) / 64
    check(x, router, 12)
    check(x, router, 1)
    check(x, router, 48)
