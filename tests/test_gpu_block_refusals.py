"""Calls of the operators around the experts that would be answered wrongly without a word
(needs an MI355X): each is refused, before any launch."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from calibration_free_moe.reader.adapters import apply_adapters
from calibration_free_moe.reader.dispatch import combine_rows, gather_rows, sort_by_expert
from calibration_free_moe.reader.norms import join_block, norm_rows

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


def test_adapters_refuse_an_out_over_their_weights():
    """Rows of `out` in memory that other tokens' products still read."""
    t = adapters()
    memory = torch.ones(4096, dtype=torch.bfloat16, device=DEVICE)
    # values 512 .. 1535, 512 .. 519 and 512 .. 515
    cases = {"encoder": memory[512:1536].view(2, 8, 64), "decoder": memory[512:1536].view(2, 64, 8),
             "slots": memory[512:520].view(torch.int32).zero_(),
             "scales": memory[512:516].view(torch.float32).fill_(1.0)}
    for name, value in cases.items():
        for out in (memory[:1024].view(4, 256)[:, :64],      # its third row begins there
                    memory[264:520].view(4, 64),             # its last row ends there
                    memory[448:1472].view(4, 256)[:, 8:72]):  # its first row ends behind
            with pytest.raises(ValueError, match="overlaps"):
                apply_adapters(**{**t, name: value}, out=out)
    # between the rows of out, and right before and behind them
    rows = torch.ones(6, 256, dtype=torch.bfloat16, device=DEVICE)
    for at in (rows[2, 64:72], rows[2, 248:], rows[0, 248:], rows[4, 64:72], rows[5, :8]):
        slots = at.view(torch.int32).zero_()
        out = rows[1:5, :64]
        out.fill_(7.0)
        apply_adapters(**{**t, "slots": slots}, out=out)
        assert bool((out == 512).all()) and bool((slots == 0).all())


def calls():
    """name -> (call, its float tensors)"""
    order = sort_by_expert(torch.zeros(4, 2, dtype=torch.int32, device=DEVICE), 2)

    def ones(*shape):
        return torch.ones(shape, device=DEVICE)

    t = adapters()
    return {
        "gather": (lambda x: gather_rows(x, order), [ones(4, 64)]),
        "combine": (lambda x, w: combine_rows(x, order, w), [ones(8, 64), ones(4, 2)]),
        "norm": (lambda x, w: norm_rows(x, w), [ones(4, 64), ones(64)]),
        "join": (lambda x, b, p, g, w: join_block(x, b, post_weight=p, gate=g, next_weight=w),
                 [ones(4, 64), ones(4, 64), ones(64), ones(4, 1), ones(64)]),
        "adapters": (lambda base, x, c, d, s: apply_adapters(base, x, c, d, t["slots"], s),
                     [t[n] for n in ("base", "hidden", "encoder", "decoder", "scales")]),
    }


NAMES = ["gather", "combine", "norm", "join", "adapters"]


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name):
    """No operator has a forward-mode derivative; a dual tensor's would be taken for zero."""
    call, tensors = calls()[name]
    with forward_ad.dual_level():
        for i, t in enumerate(tensors):
            for trained in (False, True):
                if trained and name == "adapters":
                    continue
                u = t.clone().requires_grad_(trained)
                arguments = [forward_ad.make_dual(u, torch.ones_like(t)) if j == i else v
                             for j, v in enumerate(tensors)]
                with pytest.raises(ValueError, match="forward-mode"):
                    call(*arguments)
        call(*tensors)
    call(*tensors)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("trained", [False, True])
def test_tracing_is_refused(name, trained):
    """A trace would hold the outputs' allocation and none of the kernels."""
    call, tensors = calls()[name]
    tensors = [t.clone().requires_grad_(trained and name != "adapters") for t in tensors]
    with pytest.raises(ValueError, match="torch.jit.trace"):
        torch.jit.trace(call, tuple(tensors))
    call(*tensors)


@pytest.mark.filterwarnings("ignore")
def test_tracing_the_order_is_refused():
    ids = torch.zeros(4, 2, dtype=torch.int32, device=DEVICE)
    with pytest.raises(ValueError, match="torch.jit.trace"):
        torch.jit.trace(lambda t: sort_by_expert(t, 2).places, (ids,))
    with pytest.raises(ValueError, match="torch.fx"):
        make_fx(lambda t: sort_by_expert(t, 2).places)(ids)


@pytest.mark.parametrize("name", NAMES)
def test_recording_as_torch_calls_is_refused(name):
    """Modes that look at torch's calls without recording them are none of it."""
    call, tensors = calls()[name]
    with pytest.raises(ValueError, match="torch.fx"):
        make_fx(call)(*tensors)
    want = call(*tensors)
    with FlopCounterMode(display=False):
        got = call(*tensors)
    for a, b in zip(got, want) if isinstance(want, tuple) else [(got, want)]:
        assert torch.equal(a, b)


@pytest.mark.parametrize("number", [
    1e39, -1e39, pytest.param(10 ** 400, id="long"), float("inf"), float("-inf"), float("nan")])
def test_scales_that_are_no_fp32_numbers_are_refused(number):
    x = torch.ones(2, 64, device=DEVICE)
    with pytest.raises(ValueError, match="residual_scale"):
        join_block(x, x, residual_scale=number)
    for largest in (3.4028234663852886e38, -3.4028234663852886e38, 0, 1, True):
        assert torch.equal(join_block(x, 0 * x, residual_scale=largest), x * float(largest))
