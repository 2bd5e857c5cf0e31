"""sort_by_expert, gather_rows and combine_rows against plain forms (needs an MI355X).

The order and the laid-out rows are equal; sums lie within the bounds that
block_reference derives.
"""

import pytest
import torch

from calibration_free_moe.reader.dispatch import (ExpertOrder, combine_rows, gather_rows,
                                                  sort_by_expert)
from tests import block_reference as plain

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")
TYPES = [torch.bfloat16, torch.float32]


def generator(seed):
    return torch.Generator().manual_seed(seed)


def make_ids(tokens, top_k, experts, seed, skew=False, outside=True):
    g = generator(seed)
    low, high = (-2, experts + 2) if outside else (0, experts)
    ids = torch.randint(low, high, (tokens, top_k), generator=g)
    if skew:
        ids = torch.where(torch.rand(tokens, top_k, generator=g) < 0.7, experts // 2, ids)
    return ids


def check_order(ids, experts, padding=None):
    order = sort_by_expert(ids.to(DEVICE), experts, None if padding is None else padding.to(DEVICE))
    offsets, places, pairs = plain.order(ids, experts, padding)
    assert order.offsets.tolist() == offsets
    assert order.places.flatten().tolist() == places and order.places.shape == ids.shape
    assert order.pairs.tolist() == pairs
    return order


@pytest.mark.parametrize("tokens,top_k,experts", [
    (1, 1, 1), (1, 8, 128), (2, 3, 7), (63, 1, 2), (64, 1, 64), (65, 5, 33), (131, 8, 128),
    (512, 8, 128), (513, 8, 128), (700, 8, 256), (1023, 64, 5), (40, 64, 4096), (300, 20, 1007),
    (300, 20, 1008), (900, 7, 2015), (900, 7, 2016), (900, 7, 4031), (900, 7, 4032),
    (4097, 8, 60), (40000, 7, 100), (33000, 8, 1),
])
@pytest.mark.parametrize("ids64", [False, True])
def test_order(tokens, top_k, experts, ids64):
    ids = make_ids(tokens, top_k, experts, tokens + top_k, skew=tokens % 2 == 0)
    ids = ids if ids64 else ids.int()
    check_order(ids, experts)
    check_order(ids, experts, torch.rand(tokens, generator=generator(5)) < 0.3)


def test_order_of_ids_far_outside():
    ids = torch.tensor([[2 ** 40, -2 ** 40, 3], [2 ** 32 + 1, 1, -(2 ** 63)], [2 ** 63 - 1, 0, 4]])
    check_order(ids, 4)
    check_order(torch.tensor([[2 ** 31 - 1, -2 ** 31, 0]], dtype=torch.int32), 1)


@pytest.mark.parametrize("tokens", [3, 5000])
def test_order_without_kept_pairs(tokens):
    ids = torch.full((tokens, 4), -1, dtype=torch.int32)
    check_order(ids, 9)
    check_order(torch.zeros(tokens, 4, dtype=torch.int64), 9, torch.ones(tokens, dtype=torch.bool))
    check_order(torch.full((tokens, 4), 8), 9)


def test_empty_batches():
    order = sort_by_expert(torch.empty(0, 8, dtype=torch.int32, device=DEVICE), 5)
    assert order.offsets.tolist() == [0] * 6
    x = torch.empty(0, 16, device=DEVICE, requires_grad=True)
    rows = gather_rows(x, order)
    weights = torch.empty(0, 8, device=DEVICE, requires_grad=True)
    out = combine_rows(rows, order, weights)
    assert rows.shape == out.shape == (0, 16)
    grads = torch.autograd.grad(out.sum(), (x, weights))
    assert grads[0].shape == (0, 16) and grads[1].shape == (0, 8)


SIZES = [
    # tokens, top_k, experts, hidden
    (1, 8, 128, 2048), (1, 1, 1, 1), (5, 3, 4, 7), (3, 64, 70, 24), (17, 8, 16, 512), (17, 8, 16, 520),
    (9, 9, 12, 256), (6, 17, 20, 260), (33, 2, 8, 2816), (21, 4, 8, 1001), (70, 8, 32, 64),
    (4, 2, 3, 9001), (130, 6, 64, 128), (2, 5, 6, 4096),
]


def data(tokens, top_k, experts, hidden, dtype, weights16, seed=1):
    g = generator(seed)
    ids = make_ids(tokens, top_k, experts, seed)
    padding = torch.rand(tokens, generator=g) < 0.2 if tokens > 3 else None
    x = torch.randn(tokens, hidden, generator=g).to(dtype)
    rows = torch.randn(tokens * top_k, hidden, generator=g).to(dtype)
    weights = torch.randn(tokens, top_k, generator=g).to(torch.bfloat16 if weights16 else torch.float32)
    return ids, padding, x, rows, weights


def order_of(ids, experts, padding):
    return sort_by_expert(ids.to(DEVICE), experts, None if padding is None else padding.to(DEVICE))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_gather_and_its_gradient(size, dtype):
    ids, padding, x, rows, _ = data(*size, dtype, False)
    order = order_of(ids, size[2], padding)
    places = order.places.cpu()
    leaf = x.to(DEVICE).requires_grad_()
    got = gather_rows(leaf, order)
    assert torch.equal(got.detach().cpu(), plain.gather(x, places))
    assert torch.equal(gather_rows(x.to(DEVICE), order), got)
    # dropped rows' gradients are not read
    grad = rows.clone()
    grad[(-1 - places[places < 0]).long()] = float("nan")
    (got_grad,) = torch.autograd.grad(got, leaf, grad.to(DEVICE))
    assert got_grad.dtype == dtype
    plain.within(got_grad, *plain.combine(rows, places, None))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weights16", [False, True])
def test_combine_and_its_gradients(size, dtype, weights16):
    ids, padding, x, rows, weights = data(*size, dtype, weights16)
    order = order_of(ids, size[2], padding)
    places = order.places.cpu()
    # dropped pairs' rows and weights are not read
    dropped = places < 0
    spoilt_rows, spoilt_weights = rows.clone(), weights.clone()
    spoilt_rows[(-1 - places[dropped]).long()] = float("nan")
    spoilt_weights[dropped] = float("inf")
    a, w = spoilt_rows.to(DEVICE).requires_grad_(), spoilt_weights.to(DEVICE).requires_grad_()
    out = combine_rows(a, order, w)
    assert torch.equal(combine_rows(a.detach(), order, w.detach()), out)
    plain.within(out, *plain.combine(rows, places, weights))
    grad = torch.randn(x.shape, generator=generator(9)).to(dtype)
    drows, dweights = torch.autograd.grad(out, (a, w), grad.to(DEVICE))
    want = plain.combine_backward(grad, rows, places, weights)
    assert drows.dtype == dtype and dweights.dtype == weights.dtype
    plain.within(drows, *want[:2])
    plain.within(dweights, *want[2:])
    # one gradient at a time gives the same bits
    (alone,) = torch.autograd.grad(combine_rows(a.detach(), order, w), w, grad.to(DEVICE))
    assert torch.equal(alone, dweights)
    (alone,) = torch.autograd.grad(combine_rows(a, order, w.detach()), a, grad.to(DEVICE))
    assert torch.equal(alone, drows)


def test_combine_without_weights():
    ids, padding, x, rows, _ = data(20, 5, 9, 264, torch.bfloat16, False)
    order = order_of(ids, 9, padding)
    places = order.places.cpu()
    a = rows.to(DEVICE).requires_grad_()
    out = combine_rows(a, order)
    plain.within(out, *plain.combine(rows, places, None))
    (drows,) = torch.autograd.grad(out, a, x.to(DEVICE))
    assert torch.equal(drows.cpu(), plain.gather(x, places))


def test_gradients_of_spread_outputs():
    """A gradient whose strides are zero, as that of a sum over everything."""
    ids, padding, x, rows, weights = data(12, 3, 6, 40, torch.float32, False)
    order = order_of(ids, 6, padding)
    places = order.places.cpu()
    leaf, a, w = (t.to(DEVICE).requires_grad_() for t in (x, rows, weights))
    total = gather_rows(leaf, order).sum() + combine_rows(a, order, w).sum()
    got = torch.autograd.grad(total, (leaf, a, w))
    plain.within(got[0], *plain.combine(torch.ones_like(rows), places, None))
    want = plain.combine_backward(torch.ones_like(x), rows, places, weights)
    plain.within(got[1], *want[:2])
    plain.within(got[2], *want[2:])


def test_gradients_against_differences():
    """Along random directions: the kernels' gradients and central differences of the
    64-bit form, whose own error is of the third order (none: it is bilinear)."""
    ids, padding, x, rows, weights = data(14, 4, 6, 100, torch.float32, False, seed=8)
    order = order_of(ids, 6, padding)
    places = order.places.cpu()
    leaf, a, w = (t.to(DEVICE).requires_grad_() for t in (x, rows, weights))
    g = generator(10)
    c_rows, c_out = torch.randn(rows.shape, generator=g), torch.randn(x.shape, generator=g)
    got = torch.autograd.grad((gather_rows(leaf, order), combine_rows(a, order, w)), (leaf, a, w),
                              (c_rows.to(DEVICE), c_out.to(DEVICE)))
    along = [torch.randn(t.shape, generator=g).double() for t in (x, rows, weights)]

    def loss(step):
        moved = [t.double() + step * d for t, d in zip((x, rows, weights), along)]
        first = (plain.gather(moved[0], places) * c_rows).sum()
        return first + (plain.combine(moved[1], places, moved[2])[0] * c_out).sum()

    slope = float(loss(0.5) - loss(-0.5))
    bounds = [plain.combine(c_rows, places, None)[1], *plain.combine_backward(
        c_out, rows, places, weights)[1::2]]
    allowed = sum(float((b * d.abs()).sum()) for b, d in zip(bounds, along)) + 1e-10
    assert abs(sum(float((v.cpu().double() * d).sum()) for v, d in zip(got, along)) - slope) <= allowed


def test_a_batch_without_kept_pairs():
    """All experts elsewhere: rows, sums and gradients are zeros, whatever the inputs hold."""
    order = sort_by_expert(torch.full((6, 3), -1, device=DEVICE), 4)
    x = torch.randn(6, 520, device=DEVICE, requires_grad=True)
    rows = torch.full((18, 520), float("nan"), device=DEVICE, requires_grad=True)
    weights = torch.full((6, 3), float("nan"), device=DEVICE, requires_grad=True)
    laid, out = gather_rows(x, order), combine_rows(rows, order, weights)
    grads = torch.autograd.grad((laid, out), (x, rows, weights),
                                (torch.full_like(laid, float("nan")), torch.ones_like(out)))
    for t in (laid, out, *grads):
        assert bool((t == 0).all())


def test_second_derivatives_are_refused():
    order = sort_by_expert(torch.zeros(2, 1, dtype=torch.int32, device=DEVICE), 1)
    x = torch.randn(2, 8, device=DEVICE, requires_grad=True)
    (grad,) = torch.autograd.grad((gather_rows(x, order) ** 2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        grad.sum().backward()


def test_infinities_and_nan_stay_where_they_are():
    order = sort_by_expert(torch.tensor([[0, 1], [1, 0], [2, 0]], device=DEVICE), 3)
    rows = torch.ones(6, 72, device=DEVICE)
    places = order.places
    rows[places[0, 1], 5] = float("inf")
    rows[places[1, 0], 6] = float("nan")
    out = combine_rows(rows, order, torch.full((3, 2), 0.5, device=DEVICE))
    want = torch.ones(3, 72, device=DEVICE)
    want[0, 5], want[1, 6] = float("inf"), float("nan")
    assert torch.equal(out.nan_to_num(7.0, 8.0), want.nan_to_num(7.0, 8.0))


def test_unaligned_and_sliced_rows():
    """A batch that starts inside a larger one, off a 16-byte border."""
    for dtype, h in ((torch.bfloat16, 24), (torch.float32, 12), (torch.bfloat16, 1028)):
        ids, padding, x, rows, weights = data(11, 3, 5, h, dtype, False)
        order = order_of(ids, 5, padding)
        places = order.places.cpu()
        wide = torch.empty(x.numel() + 1, dtype=dtype, device=DEVICE)[1:].view(x.shape).copy_(x)
        assert torch.equal(gather_rows(wide, order).cpu(), plain.gather(x, places))
        wide = torch.empty(rows.numel() + 1, dtype=dtype, device=DEVICE)[1:].view(rows.shape).copy_(rows)
        plain.within(combine_rows(wide, order, weights.to(DEVICE)), *plain.combine(rows, places, weights))


def test_more_values_than_32_bits_count():
    tokens, top_k, hidden = 40000, 14, 4096
    assert tokens * top_k * hidden > 2 ** 31
    ids = make_ids(tokens, top_k, 16, 3).to(DEVICE)
    order = sort_by_expert(ids, 16)
    x = torch.randn(tokens, hidden, device=DEVICE).bfloat16()
    rows = gather_rows(x, order)
    kept = int(order.offsets[-1])
    for first in range(0, tokens * top_k, 50000):
        part = rows[first:first + 50000]
        want = x[order.pairs[first:first + 50000].long() // top_k]
        want[max(0, kept - first):] = 0
        assert torch.equal(part, want)
    out = combine_rows(rows, order)
    count = (order.places >= 0).sum(1, keepdim=True)
    # sums of equal BF16 numbers are exact in FP32
    for first in range(0, tokens, 8000):
        want = (x[first:first + 8000].float() * count[first:first + 8000]).bfloat16()
        assert torch.equal(out[first:first + 8000], want)


def test_places_of_another_batch_are_skipped():
    """Places past the rows (no order holds them) are neither read nor written."""
    places = torch.tensor([[0, 100], [-100, 1]], dtype=torch.int32, device=DEVICE)
    order = ExpertOrder(torch.tensor([0, 2], dtype=torch.int32, device=DEVICE), places,
                        torch.zeros(4, dtype=torch.int32, device=DEVICE))
    x = torch.randn(2, 64, device=DEVICE)
    rows = gather_rows(x, order)
    assert torch.equal(rows[:2], x)
    out = combine_rows(rows[:2].repeat(2, 1), order)
    assert torch.equal(out, x)


def test_refusals():
    ids = torch.zeros(4, 2, dtype=torch.int32, device=DEVICE)
    order = sort_by_expert(ids, 3)
    x = torch.zeros(4, 32, device=DEVICE)
    for bad in (ids.float(), ids[0], ids.T, ids.short()):
        with pytest.raises(ValueError):
            sort_by_expert(bad, 3)
    with pytest.raises(ValueError, match="padding"):
        sort_by_expert(ids, 3, torch.zeros(3, dtype=torch.bool, device=DEVICE))
    for experts in (0, 4097):
        with pytest.raises(ValueError, match="4096"):
            sort_by_expert(ids, experts)
    for bad in (x[:3], x.half(), x.cpu(), x.T.contiguous().T, x[0]):
        with pytest.raises(ValueError):
            gather_rows(bad, order)
    rows, weights = torch.zeros(8, 32, device=DEVICE), torch.zeros(4, 2, device=DEVICE)
    for bad in (x, rows.half(), rows.T.contiguous().T):
        with pytest.raises(ValueError):
            combine_rows(bad, order, weights)
    for bad in (weights[:3], weights.half(), weights.cpu(), weights.T.contiguous().T):
        with pytest.raises(ValueError, match="weights"):
            combine_rows(rows, order, bad)
    with pytest.raises(ValueError, match="ExpertOrder"):
        gather_rows(x, ExpertOrder(order.offsets, order.places.long(), order.pairs))
    with pytest.raises(ValueError, match="ExpertOrder"):
        combine_rows(rows, ExpertOrder(order.offsets, order.places, order.pairs[:-1]))
