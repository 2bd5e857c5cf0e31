"""Calls of the operators around the experts that would be answered wrongly without a word
(needs an MI355X): each is refused, before any launch."""

import pytest
import torch

from calibration_free_moe.reader.adapters import apply_adapters

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


def adapters():
    def ones(*shape):
        return torch.ones(shape, dtype=torch.bfloat16, device=DEVICE)

    return {"base": ones(4, 64), "hidden": ones(4, 64), "encoder": ones(2, 8, 64),
            "decoder": ones(2, 64, 8), "slots": torch.zeros(4, dtype=torch.int32, device=DEVICE),
            "scales": torch.ones(2, device=DEVICE)}


@pytest.mark.parametrize("name", ["base", "hidden", "encoder", "decoder", "scales"])
def test_adapters_refuse_trained_inputs(name):
    t = adapters()
    with pytest.raises(ValueError, match="forward only"):
        apply_adapters(**{**t, name: t[name].requires_grad_()})


def test_adapters_refuse_a_trained_out():
    """Written in place it would keep the history of what it held before."""
    t = adapters()
    leaf = torch.ones(4, 64, dtype=torch.bfloat16, device=DEVICE, requires_grad=True)
    product = leaf * 2
    rows = torch.ones(4, 128, dtype=torch.bfloat16, device=DEVICE) * leaf.repeat(1, 2)
    for out in (leaf, product, rows[:, 64:]):
        before = out.detach().clone()
        with pytest.raises(ValueError, match="forward only"):
            apply_adapters(**t, out=out)
        with pytest.raises(ValueError, match="forward only"):
            apply_adapters(**{**t, "base": out.detach()}, out=out)
        assert torch.equal(out.detach(), before)
        with torch.no_grad():
            assert apply_adapters(**t, out=out) is out
            assert bool((out == 512).all())
