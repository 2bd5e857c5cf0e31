"""norm_rows and join_block against their 64-bit forms (needs an MI355X), within the
bounds that block_reference derives from the operands."""

import itertools

import pytest
import torch

from calibration_free_moe.reader.norms import join_block, norm_rows
from tests import block_reference as plain

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")
EPSILON = 1e-6
BF16, FP32 = torch.bfloat16, torch.float32


def make(tokens, size, dtype, post, gate, following, weights32=False, seed=1):
    g = torch.Generator().manual_seed(seed)
    weight_type = FP32 if weights32 else dtype
    x = torch.randn(tokens, size, generator=g)
    x[:, :: 100] *= 20
    made = {"hidden": x.to(dtype), "block": torch.randn(tokens, size, generator=g).to(dtype) / 2}
    made["post"] = (1 + torch.randn(size, generator=g) / 10).to(weight_type) if post else None
    shape = {"none": None, "channel": (size,), "row": (tokens, 1), "full": (tokens, size)}[gate]
    made["gate"] = None
    if shape:
        made["gate"] = torch.randn(shape, generator=g).to(dtype if gate == "full" else weight_type)
    made["next"] = (1 + torch.randn(size, generator=g) / 10).to(weight_type) if following else None
    return made


def call(t, scale, epsilon=EPSILON):
    out = join_block(t["hidden"], t["block"], post_weight=t["post"], gate=t["gate"],
                     residual_scale=scale, next_weight=t["next"], epsilon=epsilon)
    return out if isinstance(out, tuple) else (out, None)


def check(made, scale=1.0, epsilon=EPSILON, gradients=(True, True), seed=2):
    """Outputs and all gradients; `gradients`: which outputs the loss is made of."""
    on = {k: None if v is None else v.to(DEVICE).requires_grad_() for k, v in made.items()}
    exact = {k: None if v is None else v.double().requires_grad_() for k, v in made.items()}
    arguments = (exact["hidden"], exact["block"], exact["post"], exact["gate"],
                 float(torch.tensor(scale)), exact["next"], epsilon)
    joined, out = call(on, scale, epsilon)
    want_joined, want_out = plain.join(*arguments)
    g = torch.Generator().manual_seed(seed)
    shape, dtype = made["hidden"].shape, made["hidden"].dtype
    grads = [torch.randn(shape, generator=g).to(dtype) if wanted and o is not None else None
             for wanted, o in zip(gradients, (joined, out))]
    detached = [a.detach() if isinstance(a, torch.Tensor) else a for a in arguments]
    bounds = plain.join_bounds(*detached, *(v if v is None else v.double() for v in grads))
    plain.within(joined, want_joined.detach(), bounds["joined"])
    if out is not None:
        plain.within(out, want_out.detach(), bounds["out"])
    with torch.no_grad():
        again = call(on, scale, epsilon)
    assert torch.equal(again[0], joined) and (out is None or torch.equal(again[1], out))
    names = [k for k, v in on.items() if v is not None and k in bounds]
    pick = [i for i in range(2) if grads[i] is not None]
    got = torch.autograd.grad([(joined, out)[i] for i in pick], [on[k] for k in names],
                              [grads[i].to(DEVICE) for i in pick], retain_graph=True)
    want = torch.autograd.grad([(want_joined, want_out)[i] for i in pick],
                               [exact[k] for k in names], [grads[i].double() for i in pick])
    for name, a, b in zip(names, got, want):
        assert a.dtype == made[name].dtype, name
        plain.within(a, b, bounds[name])
    # the same bits again
    for a, b in zip(got, torch.autograd.grad([(joined, out)[i] for i in pick],
                                             [on[k] for k in names],
                                             [grads[i].to(DEVICE) for i in pick])):
        assert torch.equal(a, b)


SIZES = [1, 7, 8, 64, 65, 500, 512, 513, 520, 1001, 1024, 2048, 2049, 2056, 2816, 4096, 4097, 4104, 8192,
         8191]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_every_size(size, dtype):
    check(make(5, size, dtype, True, "channel", True), 0.7)
    check(make(3, size, dtype, False, "none", True))


@pytest.mark.parametrize("post,gate,following", list(itertools.product(
    [False, True], ["none", "channel", "row", "full"], [False, True])))
@pytest.mark.parametrize("dtype,weights32", [(BF16, False), (BF16, True), (FP32, False)])
def test_every_form(post, gate, following, dtype, weights32):
    check(make(19, 264, dtype, post, gate, following, weights32), 0.6)
    check(make(6, 77, dtype, post, gate, following, weights32))


@pytest.mark.parametrize("gradients", [(True, False), (False, True)])
@pytest.mark.parametrize("post", [False, True])
def test_a_loss_of_one_output(gradients, post):
    """The other output's gradient is none; a weight of it has none either."""
    made = make(9, 136, FP32, post, "row", True)
    if gradients[1]:
        check(made, 0.9, gradients=gradients)
        return
    on = {k: None if v is None else v.to(DEVICE).requires_grad_() for k, v in made.items()}
    joined, _ = call(on, 0.9)
    grad = torch.randn(joined.shape, generator=torch.Generator().manual_seed(3))
    names = ["hidden", "block", "gate"] + ["post"] * post
    got = torch.autograd.grad(joined, [on[k] for k in (*names, "next")], grad.to(DEVICE),
                              allow_unused=True)
    assert got[-1] is None
    exact = {k: None if v is None else v.double().requires_grad_() for k, v in made.items()}
    arguments = (exact["hidden"], exact["block"], exact["post"], exact["gate"],
                 float(torch.tensor(0.9)), None, EPSILON)
    want = torch.autograd.grad(plain.join(*arguments)[0], [exact[k] for k in names], grad.double())
    detached = [a.detach() if isinstance(a, torch.Tensor) else a for a in arguments]
    bounds = plain.join_bounds(*detached, grad.double())
    for name, a, b in zip(names, got, want):
        plain.within(a, b, bounds[name])


def check_norm(x, w, epsilon=EPSILON):
    on, weight = x.to(DEVICE).requires_grad_(), w.to(DEVICE).requires_grad_()
    out = norm_rows(on, weight, epsilon=epsilon)
    exact, exact_w = x.double().requires_grad_(), w.double().requires_grad_()
    want = plain.join(exact, None, None, None, 1.0, exact_w, epsilon)[1]
    grad = torch.randn(x.shape, generator=torch.Generator().manual_seed(4)).to(x.dtype)
    bounds = plain.join_bounds(x.double(), None, None, None, 1.0, w.double(), epsilon, None,
                               grad.double())
    plain.within(out, want.detach(), bounds["out"])
    assert torch.equal(norm_rows(on.detach(), weight.detach(), epsilon=epsilon), out)
    got = torch.autograd.grad(out, (on, weight), grad.to(DEVICE))
    wanted = torch.autograd.grad(want, (exact, exact_w), grad.double())
    assert got[0].dtype == x.dtype and got[1].dtype == w.dtype
    plain.within(got[0], wanted[0], bounds["hidden"])
    plain.within(got[1], wanted[1], bounds["next"])


@pytest.mark.parametrize("tokens", [1, 2, 255, 1023, 1024, 1025, 3001])
@pytest.mark.parametrize("dtype,weights32", [(BF16, False), (BF16, True), (FP32, False)])
def test_norm(tokens, dtype, weights32):
    made = make(tokens, 136, dtype, False, "none", True, weights32, seed=tokens)
    check_norm(made["hidden"], made["next"])


@pytest.mark.parametrize("tokens,size", [(700, 2056), (400, 4100), (1500, 520)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_more_rows_than_workgroups(tokens, size, dtype):
    """Sums over rows of which a workgroup has several, at every width of one."""
    check(make(tokens, size, dtype, True, "channel", True), 0.9)


@pytest.mark.parametrize("epsilon", [1e-30, 1e-12, 0.5, 1e30])
def test_norm_epsilon(epsilon):
    made = make(6, 200, FP32, True, "none", True)
    check_norm(made["hidden"], made["next"], epsilon)
    check(made, epsilon=epsilon)


def test_rows_of_zeros():
    """Nothing but epsilon under the root."""
    x = torch.zeros(3, 96)
    x[1] = 1.0
    w = torch.randn(96, generator=torch.Generator().manual_seed(6))
    check_norm(x, w)
    assert bool((norm_rows(x.to(DEVICE), w.to(DEVICE))[0] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("size", [40, 1000, 8192])
def test_rows_whose_squares_pass_fp32(dtype, size):
    """Magnitudes from 1e19 to 3e38 beside an ordinary row."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(5, size, generator=g).clamp(-2.5, 2.5)
    x *= torch.tensor([1.0, 1e19, 1e30, 1.2e38, 1e-25]).unsqueeze(-1)
    w = 1 + torch.randn(size, generator=g) / 10
    x, w = x.to(dtype), w.to(dtype)
    on, weight = x.to(DEVICE).requires_grad_(), w.to(DEVICE).requires_grad_()
    out = norm_rows(on, weight)
    exact, exact_w = x.double().requires_grad_(), w.double().requires_grad_()
    want = plain.join(exact, None, None, None, 1.0, exact_w, EPSILON)[1]
    grad = torch.randn(x.shape, generator=g).to(dtype)
    bounds = plain.join_bounds(x.double(), None, None, None, 1.0, w.double(), EPSILON, None,
                               grad.double())
    # one more rounding of the value times 2^-80, exact but for values that leave FP32 there
    plain.within(out, want.detach(), bounds["out"] + 2 * plain.U * want.detach().abs())
    got = torch.autograd.grad(out, (on, weight), grad.to(DEVICE))
    wanted = torch.autograd.grad(want, (exact, exact_w), grad.double())
    # gradients of large rows are subnormal in FP32: a step of 2^-149 (BF16: 2^-133)
    step = 2.0 ** -148 if dtype == FP32 else 2.0 ** -133
    plain.within(got[0], wanted[0], bounds["hidden"] + 2 * plain.U * wanted[0].abs() + step)
    plain.within(got[1], wanted[1], bounds["next"] + 2 * plain.U * grad.double().abs().sum(0) * 3)


def test_infinities_and_nan_stay_in_their_rows():
    made = make(6, 264, BF16, True, "row", True)
    made["hidden"][1, 3] = float("nan")
    made["block"][2, 4] = float("inf")
    made["hidden"][3, 5] = float("inf")
    clean = make(6, 264, BF16, True, "row", True)
    on = {k: v.to(DEVICE) for k, v in made.items()}
    joined, out = call(on, 1.0)
    want = call({k: v.to(DEVICE) for k, v in clean.items()}, 1.0)
    for got, right in ((joined, want[0]), (out, want[1])):
        assert torch.equal(got[[0, 4, 5]], right[[0, 4, 5]])
    assert bool(out[1].isnan().all()) and bool(joined[1, 3].isnan())
    assert int(joined[1].isnan().sum()) == 1
    # the norm of a row with an infinity: zero beside it, NaN in its place
    assert bool(joined[2, 4].isnan()) and int(joined[2].isnan().sum()) == 1
    assert bool(joined[3, 5].isinf()) and bool(out[3, 5].isnan())
    assert bool((out[3, :5] == 0).all()) and bool((out[3, 6:] == 0).all())


def test_gradients_against_differences():
    """Along random directions: the kernels' gradients against central differences of the
    64-bit form (1e-5 apart: their own error is about 1e-10 of the third derivative)."""
    made = make(7, 90, FP32, True, "channel", True, seed=11)
    on = {k: v.to(DEVICE).requires_grad_() for k, v in made.items()}
    g = torch.Generator().manual_seed(12)
    c = [torch.randn(7, 90, generator=g) for _ in range(2)]
    names = list(made)
    got = torch.autograd.grad(call(on, 0.5), [on[k] for k in names], [v.to(DEVICE) for v in c])
    bounds = plain.join_bounds(*(made[k].double() for k in ("hidden", "block", "post", "gate")), 0.5,
                               made["next"].double(), EPSILON, *(v.double() for v in c))
    for name, value in zip(names, got):
        along = torch.randn(made[name].shape, generator=g).double()

        def loss(step):
            t = {k: v.double() + (step * along if k == name else 0) for k, v in made.items()}
            outputs = plain.join(t["hidden"], t["block"], t["post"], t["gate"], 0.5, t["next"], EPSILON)
            return float(sum((o * v).sum() for o, v in zip(outputs, c)))

        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        allowed = float((bounds[name] * along.abs()).sum()) + 1e-6
        assert abs(float((value.cpu().double() * along).sum()) - slope) <= allowed, name


def test_gradients_of_spread_outputs():
    x = make(5, 72, FP32, False, "none", True)
    on, w = x["hidden"].to(DEVICE).requires_grad_(), x["next"].to(DEVICE).requires_grad_()
    got = torch.autograd.grad(norm_rows(on, w).sum(), (on, w))
    want = torch.autograd.grad(norm_rows(on, w), (on, w), torch.ones(5, 72, device=DEVICE))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_one_at_a_time():
    made = make(30, 264, BF16, True, "channel", True)
    grads = [torch.randn(30, 264, generator=torch.Generator().manual_seed(i)).bfloat16().to(DEVICE)
             for i in range(2)]
    on = {k: v.to(DEVICE).requires_grad_() for k, v in made.items()}
    together = torch.autograd.grad(call(on, 1.0), list(on.values()), grads)
    for name, want in zip(made, together):
        one = {k: v.to(DEVICE).requires_grad_(k == name) for k, v in made.items()}
        (got,) = torch.autograd.grad(call(one, 1.0), one[name], grads)
        assert torch.equal(got, want), name


def test_unaligned_rows_and_weights():
    for dtype, size in ((BF16, 64), (BF16, 2048), (FP32, 96)):
        made = make(4, size, dtype, True, "full", True)

        def shifted(v):
            return torch.empty(v.numel() + 1, dtype=v.dtype, device=DEVICE)[1:].view(v.shape).copy_(v)

        want = call({k: v.to(DEVICE) for k, v in made.items()}, 1.0)
        bounds = plain.join_bounds(*(made[k].double() for k in ("hidden", "block", "post", "gate")),
                                   1.0, made["next"].double(), EPSILON)
        exact = plain.join(*(made[k].double() for k in ("hidden", "block", "post", "gate")), 1.0,
                           made["next"].double(), EPSILON)
        for name in made:
            got = call({k: shifted(v) if k == name else v.to(DEVICE) for k, v in made.items()}, 1.0)
            plain.within(got[0], exact[0], bounds["joined"])
            plain.within(got[1], exact[1], bounds["out"])
        assert want[0].shape == exact[0].shape


def test_empty_batches():
    x = torch.empty(0, 64, device=DEVICE, requires_grad=True)
    w = torch.ones(64, device=DEVICE, requires_grad=True)
    joined, out = join_block(x, x.detach(), post_weight=w, next_weight=w.detach())
    assert joined.shape == out.shape == (0, 64)
    dx, dw = torch.autograd.grad(joined.sum() + out.sum(), (x, w))
    assert dx.shape == (0, 64) and bool((dw == 0).all())


def test_more_rows_than_one_grid():
    tokens = (1 << 20) + 5
    x = torch.randn(tokens, 8, device=DEVICE).bfloat16()
    w = torch.randn(8, device=DEVICE).bfloat16()
    out = norm_rows(x, w)
    assert torch.equal(out[-7:], norm_rows(x[-7:], w))
    assert torch.equal(out[:9], norm_rows(x[:9], w))


def test_more_values_than_32_bits_count():
    tokens, size = 270000, 8192
    assert tokens * size > 2 ** 31
    x = torch.empty(tokens, size, dtype=BF16, device=DEVICE).normal_()
    w = torch.randn(size, device=DEVICE).bfloat16()
    joined, out = join_block(x, x, next_weight=w)
    for part in (slice(0, 3), slice(-3, None)):
        want = join_block(x[part], x[part], next_weight=w)
        assert torch.equal(joined[part], want[0]) and torch.equal(out[part], want[1])


def test_refusals():
    x, w = torch.zeros(4, 32, device=DEVICE), torch.ones(32, device=DEVICE)
    for bad in (x.half(), x[0], x.T.contiguous().T, torch.zeros(2, 8193, device=DEVICE),
                torch.zeros(2, 0, device=DEVICE), x.double()):
        with pytest.raises(ValueError):
            norm_rows(bad, w)
    for bad in (w[:31], w.bfloat16(), w.cpu(), torch.ones(64, device=DEVICE)[::2]):
        with pytest.raises(ValueError, match="weight"):
            norm_rows(x, bad)
        with pytest.raises(ValueError, match="post_weight"):
            join_block(x, x, post_weight=bad)
        with pytest.raises(ValueError, match="next_weight"):
            join_block(x, x, next_weight=bad)
    for epsilon in (0.0, -1.0, float("nan"), float("inf"), 1e-31):
        with pytest.raises(ValueError, match="epsilon"):
            norm_rows(x, w, epsilon=epsilon)
        with pytest.raises(ValueError, match="epsilon"):
            join_block(x, x, epsilon=epsilon)
    for number in (torch.tensor(0.5), "1"):
        with pytest.raises(ValueError, match="number"):
            join_block(x, x, residual_scale=number)
        with pytest.raises(ValueError, match="number"):
            norm_rows(x, w, epsilon=number)
    for bad in (x[:3], x.bfloat16(), x.cpu()):
        with pytest.raises(ValueError, match="block"):
            join_block(x, bad)
    for bad in (w[:4], w.half(), torch.ones(3, 1, device=DEVICE), x.cpu(), torch.ones(1, 32, device=DEVICE),
                torch.ones((), device=DEVICE)):
        with pytest.raises(ValueError, match="gate"):
            join_block(x, x, gate=bad)
    with pytest.raises(ValueError, match="gate"):
        join_block(x.bfloat16(), x.bfloat16(), gate=x)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("following", [False, True])
def test_gradients_of_a_plain_sum_are_each_terms_own(dtype, following):
    """Of joined = hidden + block both terms have one gradient: sums of them, of leaves and of
    a tensor that is both terms, stay apart."""
    made = make(33, 264, dtype, False, "none", following)
    on = {k: None if v is None else v.to(DEVICE).requires_grad_() for k, v in made.items()}
    scaled = join_block(on["hidden"] * 1, on["block"] * 1, residual_scale=1,
                        next_weight=on["next"])
    outputs = scaled if following else (scaled,)
    grads = [torch.randn_like(o) for o in outputs]
    torch.autograd.backward(outputs, grads, retain_graph=True)
    assert torch.equal(on["hidden"].grad, on["block"].grad)
    one = on["hidden"].grad.clone()
    on["hidden"].grad.zero_()
    assert torch.equal(on["block"].grad, one)
    torch.autograd.backward(outputs, grads)
    assert torch.equal(on["hidden"].grad, one) and torch.equal(on["block"].grad, one + one)

    leaves = [on["hidden"].detach().requires_grad_(), on["block"].detach().requires_grad_()]
    out = join_block(*leaves, next_weight=on["next"])
    torch.autograd.backward(out if following else (out,), grads)
    leaves[0].grad.zero_()
    assert torch.equal(leaves[1].grad, one)

    both = on["hidden"].detach().requires_grad_()
    out = join_block(both, both, next_weight=on["next"])
    torch.autograd.backward(out if following else (out,), grads)
    apart = [both.detach().clone().requires_grad_() for _ in range(2)]
    out = join_block(*apart, next_weight=on["next"])
    torch.autograd.backward(out if following else (out,), grads)
    assert torch.equal(both.grad, apart[0].grad + apart[1].grad)
