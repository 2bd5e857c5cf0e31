"""apply_adapters against its 64-bit form (needs an MI355X), within the bounds that
block_reference derives from the operands."""

import pytest
import torch

from calibration_free_moe.reader.adapters import apply_adapters
from tests import block_reference as plain

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")
BF16 = torch.bfloat16


def make(tokens, hidden, outputs, adapters, rank, seed=1, runs=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g)
    x[:, :: 100] *= 20
    slots = torch.randint(-1, adapters + 1, (tokens,), generator=g)
    if runs:
        slots = slots.sort().values
    return {"base": torch.randn(tokens, outputs, generator=g).to(BF16), "hidden": x.to(BF16),
            "encoder": (torch.randn(adapters, rank, hidden, generator=g) * hidden ** -0.5).to(BF16),
            "decoder": (torch.randn(adapters, outputs, rank, generator=g) / 10).to(BF16),
            "slots": slots.int(), "scales": torch.rand(adapters, generator=g) + 0.5}


def check(made, **change):
    t = {**made, **change}
    on = {k: None if v is None else v.to(DEVICE) for k, v in t.items()}
    out = apply_adapters(**on)
    plain.within(out, *plain.adapters(**t))
    # a row whose slot names no adapter is base's, bit for bit
    slots = t["slots"].long()
    bare = (slots < 0) | (slots >= t["encoder"].shape[0])
    assert torch.equal(out.cpu()[bare].view(torch.int16), t["base"][bare].view(torch.int16))
    assert torch.equal(apply_adapters(**on), out)
    return out, on


@pytest.mark.parametrize("tokens,hidden,outputs,adapters,rank", [
    (1, 8, 8, 1, 8), (1, 2048, 2048, 8, 16), (2, 64, 72, 1, 24), (16, 128, 256, 1, 32),
    (17, 120, 264, 1, 40), (33, 264, 1000, 3, 64), (64, 2048, 512, 64, 32), (100, 1024, 320, 5, 128),
    (70, 72, 136, 2, 256), (48, 2816, 64, 7, 8), (250, 512, 96, 300, 16), (5, 1032, 8, 2, 248),
    (3, 8192, 64, 2, 16), (1024, 64, 64, 3, 16), (1023, 64, 64, 900, 8), (256, 64, 72, 9, 16),
    (256, 4104, 64, 3, 16), (7, 4096, 1032, 3, 32), (9, 4104, 1032, 3, 32), (200, 1024, 2056, 40, 40), (4, 65536, 8, 2, 8),
    (2, 8, 65536, 2, 256),
])
@pytest.mark.parametrize("scaled", [False, True])
def test_few_tokens(tokens, hidden, outputs, adapters, rank, scaled):
    made = make(tokens, hidden, outputs, adapters, rank, seed=tokens + rank)
    check(made, **({} if scaled else {"scales": None}))


@pytest.mark.parametrize("tokens,hidden,outputs,adapters,rank", [
    (1025, 64, 64, 1, 8), (1030, 128, 264, 5, 16), (1500, 264, 72, 2, 24), (1200, 512, 320, 70, 64),
    (2000, 72, 136, 3, 128), (1100, 64, 64, 4096, 8), (1400, 136, 96, 63, 40), (1300, 64, 200, 64, 256),
    (4100, 64, 64, 65, 72), (5000, 96, 64, 10, 16), (257, 64, 72, 9, 16), (300, 2048, 1024, 300, 8),
    (260, 4096, 2056, 2, 40),
])
@pytest.mark.parametrize("runs", [False, True])
def test_many_tokens(tokens, hidden, outputs, adapters, rank, runs):
    check(make(tokens, hidden, outputs, adapters, rank, seed=tokens + rank, runs=runs))


@pytest.mark.parametrize("tokens", [40, 1400])
def test_slots(tokens):
    """int64 and far outside; one adapter for all; none for any; each its own."""
    made = make(tokens, 128, 128, 6, 16)
    slots = made["slots"].long()
    check(made, slots=slots)
    check(made, slots=torch.where(slots < 0, -2 ** 40, torch.where(slots > 5, 2 ** 32 + 1, slots)))
    check(made, slots=torch.full((tokens,), 3, dtype=torch.int32))
    out, on = check(made, slots=torch.full((tokens,), -1, dtype=torch.int32))
    assert torch.equal(out, on["base"])
    many = make(tokens, 64, 64, tokens, 8)
    check(many, slots=torch.randperm(tokens, generator=torch.Generator().manual_seed(2)))


@pytest.mark.parametrize("tokens", [30, 1300])
def test_in_place_and_slices(tokens):
    """base, hidden and out as columns of wider rows; out as base; rows beside them stay."""
    made = make(tokens, 128, 192, 4, 24)
    want = apply_adapters(**{k: v.to(DEVICE) for k, v in made.items()})
    wide = torch.full((tokens, 400), 7.0, dtype=BF16, device=DEVICE)
    base, x = wide[:, 8:200], wide[:, 208:336]
    base.copy_(made["base"])
    x.copy_(made["hidden"])
    rest = {k: made[k].to(DEVICE) for k in ("encoder", "decoder", "slots", "scales")}
    before = wide.clone()
    assert torch.equal(apply_adapters(base, x, **rest), want)
    assert torch.equal(wide, before)
    out = torch.full((tokens, 256), 5.0, dtype=BF16, device=DEVICE)
    assert apply_adapters(base, x, **rest, out=out[:, 64:]).data_ptr() == out[:, 64:].data_ptr()
    assert torch.equal(out[:, 64:], want) and bool((out[:, :64] == 5).all())
    got = apply_adapters(base, x, **rest, out=base)
    assert got is base and torch.equal(base, want)
    before[:, 8:200] = want
    assert torch.equal(wide, before)


def test_out_is_hidden():
    for tokens in (9, 1200):
        made = make(tokens, 128, 128, 3, 16)
        on = {k: v.to(DEVICE) for k, v in made.items()}
        want = apply_adapters(**on)
        assert torch.equal(apply_adapters(**on, out=on["hidden"]), want)


def test_rows_of_one_base():
    """A base that is one row for all tokens (stride zero)."""
    made = make(20, 64, 64, 2, 8)
    base = made["base"][:1].to(DEVICE).expand(20, 64)
    on = {k: v.to(DEVICE) for k, v in made.items() if k != "base"}
    out = apply_adapters(base, **on)
    plain.within(out, *plain.adapters(**{**made, "base": made["base"][:1].expand(20, 64)}))


def test_zeros_of_either_sign_and_nan_of_bare_rows():
    made = make(6, 64, 64, 2, 8)
    made["base"][0] = -0.0
    made["base"][1].view(torch.int16).fill_(0x7F81)
    made["slots"] = torch.tensor([-1, 5, -1, 0, 1, 2], dtype=torch.int32)
    check_bits = apply_adapters(**{k: v.to(DEVICE) for k, v in made.items()}).cpu()
    for t in (0, 1, 2, 5):
        assert torch.equal(check_bits[t].view(torch.int16), made["base"][t].view(torch.int16))


@pytest.mark.parametrize("tokens", [20, 1200])
def test_infinities_and_nan_stay_in_their_rows(tokens):
    made = make(tokens, 128, 64, 3, 16)
    made["slots"] = (torch.arange(tokens) % 3).int()
    on = {k: v.to(DEVICE) for k, v in made.items()}
    want = apply_adapters(**on)
    on["hidden"][3, 7], on["hidden"][7, 70] = float("nan"), float("inf")
    on["base"][5, 2] = float("nan")
    out = apply_adapters(**on)
    others = [t for t in range(tokens) if t not in (3, 5, 7)]
    assert torch.equal(out[others], want[others])
    assert bool(out[3].isnan().all()) and not bool(out[7].isfinite().any())
    assert bool(out[5, 2].isnan()) and int(out[5].isnan().sum()) == 1
    # an infinite weight makes infinities of its adapter's tokens, not NaN
    made["decoder"][1, 9, 4] = float("inf")
    out = apply_adapters(**{k: v.to(DEVICE) for k, v in made.items()})
    assert bool(out[1::3, 9].isinf().all())
    out[1::3, 9] = want[1::3, 9]
    assert torch.equal(out, want)


@pytest.mark.parametrize("tokens", [3, 300])
def test_infinite_weights_and_inner_values_of_any_kind(tokens):
    """Inner values that are BF16 numbers themselves, and infinite ones: infinities where the
    sum has one, not NaN."""
    made = make(tokens, 64, 64, 1, 8)
    made["slots"][:] = 0
    made["hidden"][:] = 0
    made["hidden"][:, 5] = 0.5
    made["encoder"][:] = 0
    made["encoder"][0, :, 5] = 1.0
    made["decoder"][0, 3, 2], made["decoder"][0, 4, 2] = float("inf"), float("-inf")
    out = apply_adapters(**{k: v.to(DEVICE) for k, v in made.items()}).cpu()
    assert bool((out[:, 3] == float("inf")).all()) and bool((out[:, 4] == float("-inf")).all())
    assert bool(out[:, 5:].isfinite().all())
    made = make(tokens, 64, 64, 1, 8)
    made["slots"][:] = 0
    made["hidden"][0, 5] = float("inf")
    made["encoder"][0] = made["encoder"][0].abs() + 0.01
    made["decoder"] = made["decoder"].abs() + 0.01
    out = apply_adapters(**{k: v.to(DEVICE) for k, v in made.items()}).cpu()
    assert bool((out[0] == float("inf")).all()) and bool(out[1:].isfinite().all())


def test_the_batch_does_not_matter():
    """A token alone and among others: the same value to the order of the sums."""
    made = make(40, 256, 128, 4, 32)
    on = {k: v.to(DEVICE) for k, v in made.items()}
    out = apply_adapters(**on)
    for t in (0, 13, 39):
        alone = {k: on[k][t:t + 1] if k in ("base", "hidden", "slots") else on[k] for k in on}
        assert torch.equal(apply_adapters(**alone)[0], out[t])


@pytest.mark.parametrize("tokens", [2, 300])
def test_more_weights_than_32_bits_count(tokens):
    """The last of many adapters, 5 GB of either weight, as the only one of a short list."""
    n, rank, size = 300, 128, 65536
    assert n * rank * size > 2 ** 31
    g = torch.Generator(device=DEVICE).manual_seed(3)
    x = torch.randn(tokens, size, generator=g, device=DEVICE).bfloat16()
    base = torch.randn(tokens, size, generator=g, device=DEVICE).bfloat16()
    encoder = torch.empty(n, rank, size, dtype=BF16, device=DEVICE)
    decoder = torch.empty(n, size, rank, dtype=BF16, device=DEVICE)
    encoder[-1] = (torch.randn(rank, size, generator=g, device=DEVICE) / 256).bfloat16()
    decoder[-1] = torch.randn(size, rank, generator=g, device=DEVICE).bfloat16()
    slots = torch.full((tokens,), n - 1, dtype=torch.int32, device=DEVICE)
    got = apply_adapters(base, x, encoder, decoder, slots)
    want = apply_adapters(base, x, encoder[-1:].clone(), decoder[-1:].clone(), torch.zeros_like(slots))
    assert torch.equal(got, want) and not torch.equal(got, base)


def test_empty_batches():
    made = make(3, 64, 64, 2, 8)
    on = {k: v.to(DEVICE) for k, v in made.items()}
    out = apply_adapters(**{k: on[k][:0] if k in ("base", "hidden", "slots") else on[k] for k in on})
    assert out.shape == (0, 64)


def test_refusals():
    made = make(4, 64, 72, 2, 16)
    on = {k: v.to(DEVICE) for k, v in made.items()}

    def refuse(match=None, **change):
        with pytest.raises(ValueError, match=match):
            apply_adapters(**{**on, **change})

    refuse(hidden=on["hidden"].float())
    refuse(hidden=on["hidden"][:3])
    refuse(hidden=on["hidden"].cpu())
    refuse(hidden=on["hidden"].T.contiguous().T)
    refuse(hidden=torch.zeros(4, 70, dtype=BF16, device=DEVICE)[:, :64])
    refuse(hidden=torch.zeros(4, 72, dtype=BF16, device=DEVICE)[:, 4:68])
    refuse(base=on["base"][:, :64])
    refuse(encoder=on["encoder"].transpose(1, 2).contiguous().transpose(1, 2))
    refuse(encoder=on["encoder"][:, :8])
    refuse(decoder=on["decoder"].half())
    refuse(slots=on["slots"].short())
    refuse(slots=on["slots"][:3])
    refuse(scales=on["scales"].bfloat16())
    refuse(scales=on["scales"][:1])
    refuse("multiples of 8", base=on["base"][:, :68], decoder=on["decoder"][:, :68].contiguous())
    refuse("rank", encoder=on["encoder"][:, :12].contiguous(), decoder=on["decoder"][..., :12].contiguous())
    refuse("out must", out=torch.zeros(4, 64, dtype=BF16, device=DEVICE))
    refuse("out must", out=torch.zeros(1, 72, dtype=BF16, device=DEVICE).expand(4, 72))
    wide = torch.zeros(5, 160, dtype=BF16, device=DEVICE)
    refuse("overlaps", base=wide[:4, :72], out=wide[1:, :72])
    refuse("overlaps", base=wide[:4, :72], out=wide[:4, 64:136])
    refuse("overlaps", hidden=wide[:4, :64], out=wide[:4, 8:80])
    refuse("forward only", hidden=on["hidden"].clone().requires_grad_())
    refuse("forward only", decoder=on["decoder"].clone().requires_grad_())
    with torch.no_grad():
        apply_adapters(**{**on, "hidden": on["hidden"].clone().requires_grad_()})


def test_out_saved_for_a_backward_pass_is_seen_to_have_changed():
    made = make(20, 64, 64, 2, 8)
    on = {k: v.to(DEVICE) for k, v in made.items()}
    factor = torch.ones(64, device=DEVICE, dtype=BF16, requires_grad=True)
    product = on["base"] * factor
    apply_adapters(**on)
    (product * 1).sum().backward(retain_graph=True)
    apply_adapters(**on, out=on["base"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        base = on["base"].clone()
        apply_adapters(**{**on, "base": base}, out=base)


@pytest.mark.parametrize("tokens,hidden,outputs,adapters,rank", [
    (1024, 64, 64, 3, 32), (512, 64, 1032, 4, 24), (513, 64, 1032, 4, 24), (700, 64, 64, 460, 8),
    (700, 64, 64, 500, 8), (900, 4096, 264, 180, 32), (900, 4096, 264, 300, 32), (1000, 72, 1024, 1, 16),
    (257, 2048, 4096, 8, 16), (64, 512, 8192, 64, 16), (64, 512, 8200, 64, 16), (16, 64, 65536, 2, 8),
])
@pytest.mark.parametrize("ids64", [False, True])
def test_sizes_at_which_the_launches_change(tokens, hidden, outputs, adapters, rank, ids64):
    made = make(tokens, hidden, outputs, adapters, rank, seed=tokens + rank)
    check(made, **({"slots": made["slots"].long()} if ids64 else {}))


@pytest.mark.parametrize("tokens", [257, 700, 1024])
def test_out_is_hidden_of_few_ranks(tokens):
    made = make(tokens, 128, 128, 3, 16)
    on = {k: v.to(DEVICE) for k, v in made.items()}
    want = check(made)[0]
    got = apply_adapters(**on, out=on["hidden"])
    plain.within(got, *plain.adapters(**made))
    assert torch.equal(got.isnan(), want.isnan())
