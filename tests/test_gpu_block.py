"""A block from its norm to the next one's, as a prompt and a training step run it: norm,
router, rows by expert, the experts' products, back, adapters beside a shared expert's
projection, and the join (needs an MI355X). Also on side streams, two calls at once, and in
replayed graphs."""

import pytest
import torch

from calibration_free_moe.reader.adapters import apply_adapters
from calibration_free_moe.reader.dispatch import combine_rows, gather_rows, sort_by_expert
from calibration_free_moe.reader.experts import routed_experts
from calibration_free_moe.reader.norms import join_block, norm_rows
from calibration_free_moe.reader.progressive import channel_major_down
from calibration_free_moe.reader.router import route
from tests import block_reference as plain
from tests import layer_reference
from tests.synthetic import make_layer

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


def products(rows, offsets, gate_up, down):
    """Expert after expert, in FP32, from offsets on the host."""
    ends = offsets.tolist()
    parts = []
    for e, (first, last) in enumerate(zip(ends, ends[1:])):
        both = rows[first:last].float() @ gate_up[e].float().T
        gate, up = both.chunk(2, dim=-1)
        parts.append((torch.nn.functional.silu(gate) * up) @ down[e].float().T)
    parts.append(rows[ends[-1]:].float() * 0)
    return torch.cat(parts)


@pytest.mark.parametrize("tokens", [1, 6, 40, 700])
def test_rows_by_expert_are_the_whole_layer(tokens):
    """norm, route, rows, products and back agree with routed_experts on the same rows."""
    layer = make_layer(hidden=256, width=128, experts=16, top_k=4, rank=16, tokens=tokens, seed=31)
    weight = (1 + torch.arange(256) / 1000).bfloat16()
    x = norm_rows(layer.hidden.to(DEVICE), weight.to(DEVICE))
    gate_up, down = layer.gate_up.to(DEVICE), layer.down.to(DEVICE)
    padding = torch.zeros(tokens, dtype=torch.bool)
    if tokens > 3:
        padding[-2:] = True
    ids, weights = route(x, layer.router.to(DEVICE), 4)
    order = sort_by_expert(ids, 16, padding.to(DEVICE))
    out = combine_rows(products(gather_rows(x, order), order.offsets, gate_up, down), order, weights)
    whole = routed_experts(x, gate_up, channel_major_down(down), ids, weights, padding.to(DEVICE))
    want, bound = layer_reference.layer(x.cpu(), layer.gate_up, layer.down, ids.cpu(), weights, padding)
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    assert bool(((whole.cpu().double() - want).abs() <= bound).all())


def step(x, block, ids, weights, norms, gate, base, encoder, decoder, slots):
    """One pass through every operator; a stand-in product between rows and back."""
    order = sort_by_expert(ids, 8)
    rows = gather_rows(norm_rows(x, norms[0]), order)
    mixed = combine_rows(rows, order, weights)
    shared = apply_adapters(base, x.detach(), encoder, decoder, slots)
    joined, following = join_block(x, block + mixed, post_weight=norms[1], gate=gate,
                                   residual_scale=0.5, next_weight=norms[2])
    return joined, following, shared, order.offsets, order.places


def inputs(tokens, seed, leaves=False):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g).bfloat16().to(DEVICE)

    x, block = normal(tokens, 192), normal(tokens, 192)
    ids = torch.randint(-1, 8, (tokens, 3), generator=g).to(DEVICE)
    weights = torch.rand(tokens, 3, generator=g).to(DEVICE)
    norms = [normal(192) for _ in range(3)]
    gate = torch.rand(tokens, 1, generator=g).to(DEVICE)
    rest = (normal(tokens, 64), normal(4, 16, 192), normal(4, 64, 16),
            torch.randint(-1, 4, (tokens,), generator=g).to(DEVICE))
    if leaves:
        for t in (x, block, weights, gate, *norms):
            t.requires_grad_()
    return x, block, ids, weights, norms, gate, *rest


def test_gradients_through_the_operators():
    """The chain's gradients are those of the 64-bit chain, FP32 rows: relative 1e-4 of the
    largest (each operator's own bound, at most 1e-5 of it here, passed on by the next)."""
    x, block, ids, weights, norms, gate, *_ = inputs(30, 1)
    leaves = [t.float().requires_grad_() for t in (x, block, weights, *norms, gate)]
    x, block, weights, first, post, following, gate = leaves
    order = sort_by_expert(ids, 8)
    mixed = combine_rows(gather_rows(norm_rows(x, first), order) ** 2, order, weights)
    joined, out = join_block(x, block + mixed, post_weight=post, gate=gate, residual_scale=0.5,
                             next_weight=following)
    g = torch.Generator().manual_seed(5)
    c = [torch.randn(30, 192, generator=g) for _ in range(2)]
    got = torch.autograd.grad((joined, out), leaves, [v.to(DEVICE) for v in c])
    exact = [t.detach().cpu().double().requires_grad_() for t in leaves]
    x, block, weights, first, post, following, gate = exact
    normed = plain.join(x, None, None, None, 1.0, first, 1e-6)[1]
    kept = (ids.cpu() >= 0).unsqueeze(-1)
    mixed = (normed.unsqueeze(1) ** 2 * weights.unsqueeze(-1) * kept).sum(1)
    outputs = plain.join(x, block + mixed, post, gate, 0.5, following, 1e-6)
    want = torch.autograd.grad(outputs, exact, [v.double() for v in c])
    for a, b in zip(got, want):
        assert float((a.cpu().double() - b).abs().max()) <= 1e-4 * float(b.abs().max())


@pytest.mark.parametrize("tokens", [1, 50, 1500])
def test_two_streams_at_once(tokens):
    calls = [inputs(tokens, 1), inputs(tokens, 2)]
    want = [step(*call) for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(5):
        for i, (stream, call) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(stream):
                got[i].append(step(*call))
    torch.cuda.synchronize()
    for results, right in zip(got, want):
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, right))


@pytest.mark.parametrize("tokens", [1, 50, 1500])
def test_replayed_graphs(tokens):
    """Two graphs replayed in turn with new rows and eager work between; every replay
    equals an eager call, bit for bit."""
    held = [inputs(tokens, 1), inputs(tokens, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for call in held:
            step(*call)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for call in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*call))
        graphs.append(graph)
    for seed in range(3, 7):
        fresh = [inputs(tokens, seed), inputs(tokens, seed + 10)]
        for call, new in zip(held, fresh):
            for old, value in zip(call, new):
                for a, b in zip(*((old, value) if isinstance(old, list) else ([old], [value]))):
                    a.copy_(b)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, new in zip(outs, fresh):
            assert all(torch.equal(a, b) for a, b in zip(out, step(*new)))


def gradients(call):
    x, block, _, weights, norms, gate, *_ = call
    joined, following, *_ = step(*call)
    return torch.autograd.grad((joined, following), (x, block, weights, *norms, gate),
                               (torch.ones_like(joined), torch.ones_like(following)))


def test_a_captured_training_step():
    """Forward and backward in one graph, its leaves in no eager graph; replays with new
    values equal eager gradients of other leaves, bit for bit."""
    warm = inputs(40, 1, leaves=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gradients(warm)
    torch.cuda.current_stream().wait_stream(side)
    held = inputs(40, 2, leaves=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gradients(held)
    for seed in (3, 4, 5):
        fresh = inputs(40, seed, leaves=True)
        with torch.no_grad():
            for old, value in zip(held, fresh):
                for a, b in zip(*((old, value) if isinstance(old, list) else ([old], [value]))):
                    a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, gradients(fresh)))
