"""The operators' nodes in torch's autograd engine (needs an MI355X): what a training program
does with a graph besides one backward pass. Each result is that of the plain pass, bit for bit."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from calibration_free_moe.reader import _ext
from calibration_free_moe.reader.dispatch import combine_rows, gather_rows, sort_by_expert
from calibration_free_moe.reader.norms import join_block, norm_rows

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


def numbers(*shape, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(DEVICE)


def operators():
    """name -> (call, its tensors)"""
    ids = torch.randint(-1, 6, (9, 3), generator=torch.Generator().manual_seed(3)).to(DEVICE)
    order = sort_by_expert(ids, 5)
    x, b, w = numbers(9, 136), numbers(9, 136, seed=2), numbers(136, seed=4)
    return {
        "gather": (lambda x: gather_rows(x, order), (x,)),
        "combine": (lambda rows, weights: combine_rows(rows, order, weights),
                    (numbers(27, 136), numbers(9, 3, seed=5))),
        "sum": (lambda rows: combine_rows(rows, order), (numbers(27, 136),)),
        "norm": (lambda x, w: norm_rows(x, w), (x, w)),
        "join": (lambda x, b: join_block(x, b), (x, b)),
        "join-next": (lambda x, b, w: join_block(x, b, next_weight=w), (x, b, w)),
        "join-all": (lambda x, b, p, g, w: join_block(
            x, b, post_weight=p, gate=g, residual_scale=0.7, next_weight=w),
            (x, b, numbers(136, seed=6), numbers(9, 1, seed=7), w)),
    }


NAMES = ["gather", "combine", "sum", "norm", "join", "join-next", "join-all"]


def setup(name):
    call, tensors = operators()[name]
    return call, [t.clone().requires_grad_() for t in tensors]


def outputs(result):
    return result if isinstance(result, tuple) else (result,)


def along(result):
    return [numbers(*o.shape, seed=9 + i) for i, o in enumerate(outputs(result))]


def gradients(call, leaves, **options):
    result = call(*leaves)
    return torch.autograd.grad(outputs(result), leaves, along(result), **options)


def same(got, want):
    return len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES)
def test_graphs_kept_freed_and_differentiable(name):
    call, leaves = setup(name)
    want = gradients(call, leaves)
    result = call(*leaves)
    to = along(result)
    assert all(o.requires_grad and o.grad_fn is not None for o in outputs(result))
    for _ in range(2):
        assert same(torch.autograd.grad(outputs(result), leaves, to, retain_graph=True), want)
    assert same(torch.autograd.grad(outputs(result), leaves, to), want)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(outputs(result), leaves, to)
    got = gradients(call, leaves, create_graph=True)
    assert same([g.detach() for g in got], want)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        sum(g.sum() for g in got).backward()


@pytest.mark.parametrize("name", NAMES)
def test_each_gradient_alone(name):
    call, leaves = setup(name)
    want = gradients(call, leaves)
    for i, t in enumerate(leaves):
        alone = [u.detach().requires_grad_(j == i) for j, u in enumerate(leaves)]
        result = call(*alone)
        assert same(torch.autograd.grad(outputs(result), alone[i], along(result)), want[i:i + 1])
        # asked for alone, of a graph that has all
        result = call(*leaves)
        assert same(torch.autograd.grad(outputs(result), t, along(result)), want[i:i + 1])


@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors(name):
    """Kept on the host, packed and unpacked, or seen to have changed."""
    call, leaves = setup(name)
    want = gradients(call, leaves)
    with torch.autograd.graph.save_on_cpu():
        result = call(*leaves)
    assert same(torch.autograd.grad(outputs(result), leaves, along(result)), want)
    result = call(*leaves)
    to = along(result)
    with torch.no_grad():
        leaves[0].add_(1)
    if name in ("gather", "sum"):  # whose gradients are of the order alone
        assert same(torch.autograd.grad(outputs(result), leaves, to), want)
        return
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(outputs(result), leaves, to)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_passes(name, reentrant):
    call, leaves = setup(name)
    want = gradients(call, leaves)
    result = checkpoint(call, *leaves, use_reentrant=reentrant)
    torch.autograd.backward(outputs(result), along(result))
    assert same([t.grad for t in leaves], want)


@pytest.mark.parametrize("name", NAMES)
def test_threads_streams_and_anomalies(name):
    call, leaves = setup(name)
    want = gradients(call, leaves)
    with torch.autograd.set_multithreading_enabled(False):
        assert same(gradients(call, leaves), want)
    with torch.autograd.detect_anomaly(check_nan=True):
        assert same(gradients(call, leaves), want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = gradients(call, leaves)
    stream.synchronize()
    assert same(got, want)


def test_refusals_are_errors_of_the_call():
    """A size that the C entry refuses ends neither a thread nor the process."""
    wide = torch.zeros(2, 8200, device=DEVICE, requires_grad=True)
    weight = torch.ones(8200, device=DEVICE)
    with pytest.raises(ValueError, match="1 to 8192"):
        _ext.operators().join_block(wide, None, None, None, weight, 1.0, 1e-6, _ext.FP32)


def test_rows_are_kept_for_the_weights_gradient_alone():
    order = sort_by_expert(torch.zeros(64, 2, dtype=torch.int32, device=DEVICE), 1)
    weights = numbers(64, 2)
    for trained in (False, True):
        rows = numbers(128, 2048).requires_grad_()
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.shape) or t, lambda t: t):
            combine_rows(rows, order, weights.detach().requires_grad_(trained))
        assert (rows.shape in kept) == trained
