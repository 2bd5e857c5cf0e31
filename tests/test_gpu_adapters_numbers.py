"""The numbers inside apply_adapters (needs an MI355X): sums whose 64-bit value is known exactly."""

import pytest
import torch

from calibration_free_moe.reader.adapters import apply_adapters

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")
BF16 = torch.bfloat16

# (tokens, hidden, outputs, adapters, rank): both products in one launch, in two, and sorted
SHAPES = [(1, 64, 64, 1, 8), (20, 2048, 72, 2, 32), (300, 264, 136, 3, 16), (20, 512, 72, 2, 40),
          (100, 4104, 64, 3, 256), (600, 264, 136, 3, 72), (1100, 512, 72, 2, 8), (2000, 2056, 264, 4, 128)]


def zeros(tokens, hidden, outputs, adapters, rank):
    return {"base": torch.zeros(tokens, outputs, dtype=BF16),
            "hidden": torch.zeros(tokens, hidden, dtype=BF16),
            "encoder": torch.zeros(adapters, rank, hidden, dtype=BF16),
            "decoder": torch.zeros(adapters, outputs, rank, dtype=BF16),
            "slots": (torch.arange(tokens) % adapters).int()}


@pytest.mark.parametrize("shape", SHAPES)
def test_inner_values_are_held_in_24_bits(shape):
    """Two inner values, 1 + 2^-9 + 2^-20 + 2^-23 and 1 + 2^-9 (every partial sum of which is
    an FP32 number), and an output that is their difference: 1.125 2^-20, a BF16 number. All
    of it is exact, so that nothing but bits left out of an inner value can change it."""
    tokens, hidden, outputs, adapters, rank = shape
    t = zeros(*shape)
    columns = [0, hidden // 3, hidden // 2, hidden - 1]
    size = 2.0 ** torch.randint(-3, 4, (tokens, 1), generator=torch.Generator().manual_seed(1))
    size *= 1 - 2 * (torch.arange(tokens) % 2).unsqueeze(-1)
    t["hidden"][:, columns] = (size * torch.tensor([1, 2.0 ** -9, 2.0 ** -20, 2.0 ** -23])).to(BF16)
    weight = 2.0 ** (torch.arange(outputs) % 5 - 2) * (1 - 2 * (torch.arange(outputs) % 3 % 2))
    for a in range(adapters):
        whole, short = (3 * a) % (rank - 1), rank - 1
        t["encoder"][a, whole, columns] = 1
        t["encoder"][a, short, columns[:2]] = 1
        t["decoder"][a, :, whole], t["decoder"][a, :, short] = weight.to(BF16), -weight.to(BF16)
    out = apply_adapters(**{k: v.to(DEVICE) for k, v in t.items()})
    want = size * weight * 1.125 * 2.0 ** -20
    assert torch.equal(want.to(BF16).float(), want.float())
    assert torch.equal(out.cpu(), want.to(BF16))


@pytest.mark.parametrize("shape", SHAPES)
def test_infinite_weights_of_small_inner_values(shape):
    """Infinite where the product is, with no zero part that would make it NaN."""
    tokens, hidden, outputs, adapters, rank = shape
    t = zeros(*shape)
    t["hidden"][:, 1], t["hidden"][:, hidden - 2] = 2.0 ** -60, 2.0 ** -80
    t["encoder"][:, :, 1], t["encoder"][:, :, hidden - 2] = 2.0 ** -20, 2.0 ** -20
    t["encoder"][:, 0] *= -1
    t["decoder"][:, 3, 0], t["decoder"][:, 5, rank - 1] = float("inf"), float("inf")
    out = apply_adapters(**{k: v.to(DEVICE) for k, v in t.items()}).cpu()
    assert bool((out[:, 3] == -float("inf")).all()) and bool((out[:, 5] == float("inf")).all())
    out[:, [3, 5]] = 0
    assert bool((out == 0).all())


@pytest.mark.parametrize("shape", SHAPES)
def test_scales_apply_to_whole_inner_values(shape):
    """Inner values of terms that cancel to 1 before a scale of 2^110, which would take the
    terms out of FP32: 2^110, times weights of 2^-110."""
    tokens, hidden, outputs, adapters, rank = shape
    t = zeros(*shape)
    t["hidden"][:, 0], t["hidden"][:, hidden - 1], t["hidden"][:, hidden // 2] = 2.0 ** 20, -2.0 ** 20, 1
    t["encoder"][:] = 1
    t["decoder"][:, :, 0] = 2.0 ** -110
    t["scales"] = torch.full((adapters,), 2.0 ** 110)
    out = apply_adapters(**{k: v.to(DEVICE) for k, v in t.items()}).cpu()
    assert bool((out == 1).all())


@pytest.mark.parametrize("shape", SHAPES)
def test_infinite_scales(shape):
    """Of hidden values that are zero but in one place."""
    t = zeros(*shape)
    t["hidden"][:, 0] = 1
    t["encoder"][:], t["decoder"][:] = 1, 1
    t["scales"] = torch.full((shape[3],), float("inf"))
    out = apply_adapters(**{k: v.to(DEVICE) for k, v in t.items()}).cpu()
    assert bool((out == float("inf")).all())


@pytest.mark.parametrize("tokens", [9, 257, 700, 1024, 1100])
def test_out_is_hidden_beside_nan_and_infinities(tokens):
    """Rows with a NaN or an infinity stay alone where each token's rows are read and written."""
    g = torch.Generator().manual_seed(tokens)
    t = {"base": torch.randn(tokens, 128, generator=g).to(BF16),
         "hidden": torch.randn(tokens, 128, generator=g).to(BF16),
         "encoder": (torch.randn(3, 16, 128, generator=g) / 11).to(BF16),
         "decoder": torch.randn(3, 128, 16, generator=g).to(BF16),
         "slots": torch.arange(tokens) % 3}
    clean = apply_adapters(**{k: v.to(DEVICE) for k, v in t.items()})
    t["hidden"][2, 7], t["hidden"][5, 70] = float("nan"), float("inf")
    t["base"][8, 3] = float("nan")
    on = {k: v.to(DEVICE) for k, v in t.items()}
    apart = apply_adapters(**on)
    assert apply_adapters(**on, out=on["hidden"]) is on["hidden"]
    mask = torch.zeros(tokens, 128, dtype=torch.bool, device=DEVICE)
    mask[2], mask[8, 3] = True, True
    for out in (apart, on["hidden"]):
        assert torch.equal(out[:5].isnan(), mask[:5]) and torch.equal(out[6:].isnan(), mask[6:])
        assert not bool(out[5].isfinite().any())
        others = ~mask
        others[5] = False
        assert torch.equal(out[others], clean[others])
