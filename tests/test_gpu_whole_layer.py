"""route, quantise_fp4 and routed_experts in a row, as a decode step runs them
(needs an MI355X): against the float64 layer, beside a ProgressiveReader over the
same weights, on side streams, and captured in graphs that are replayed.
"""

import pytest
import torch

from calibration_free_moe.reader.budget import compile_budget
from calibration_free_moe.reader.experts import routed_experts
from calibration_free_moe.reader.microscale import dequantise_fp4, quantise_fp4
from calibration_free_moe.reader.progressive import ProgressiveReader, channel_major_down
from calibration_free_moe.reader.router import route
from tests import layer_reference as plain
from tests.synthetic import make_layer

pytestmark = pytest.mark.gpu

DEVICE = torch.device("cuda:0")


def weights_of(layer, fp4):
    gate_up, down = layer.gate_up.to(DEVICE), layer.down.to(DEVICE)
    if fp4:
        return quantise_fp4(gate_up), quantise_fp4(down)
    return gate_up, channel_major_down(down)


@pytest.mark.parametrize("fp4", [False, True], ids=["bf16", "fp4"])
@pytest.mark.parametrize("tokens", [1, 6, 40])
def test_route_then_experts(tokens, fp4):
    layer = make_layer(hidden=512, width=256, experts=16, top_k=4, rank=16, tokens=tokens, seed=31)
    x, router = layer.hidden.to(DEVICE), layer.router.to(DEVICE)
    gate_up, down = weights_of(layer, fp4)
    ids, weights = route(x, router, 4)
    got = routed_experts(x, gate_up, down, ids, weights).cpu().double()
    want_ids, _, _ = plain.routing(layer.hidden, layer.router, 4)
    assert torch.equal(ids.cpu().long(), want_ids)
    values = (layer.gate_up, layer.down)
    if fp4:
        values = tuple(plain.quantised(w)[2] for w in values)
    want, bound = plain.layer(layer.hidden, *values, ids, weights)
    assert bool(((got - want).abs() <= bound).all())


def test_the_readers_own_weights_and_routing():
    """A reader and the whole layer share borrowed weights, ids and weights; a plan
    that keeps every channel is the same layer. It rounds to BF16 after each step, so
    the two agree within the reader's own bound, 1e-2 of the layer's norm."""
    layer = make_layer(hidden=512, width=256, experts=8, top_k=4, rank=16, tokens=5, seed=32)
    gate_up, down = weights_of(layer, False)
    plan = compile_budget(hidden_size=512, expert_width=256, top_k=4, retention=1.0,
                          screen_keep=1.0)
    reader = ProgressiveReader(gate_up, down, layer.encoder.to(DEVICE), layer.decoder.to(DEVICE),
                               plan, 5, selection_score="point")
    x = layer.hidden.to(DEVICE)
    ids, weights = route(x, layer.router.to(DEVICE), 4)
    sparse = reader(x, ids, weights).cpu().double()
    dense = routed_experts(x, reader.native_gu, reader.down, ids, weights).cpu().double()
    want, bound = plain.layer(layer.hidden, layer.gate_up, layer.down, ids, weights)
    assert bool(((dense - want).abs() <= bound).all())
    assert float((dense - sparse).norm()) <= 1e-2 * float(dense.norm())


def test_a_shared_expert_is_a_layer_of_one():
    layer = make_layer(hidden=256, width=128, experts=1, top_k=1, rank=16, tokens=7, seed=33)
    gate_up, down = weights_of(layer, False)
    gate = torch.rand(7, 1, generator=torch.Generator().manual_seed(1))
    ids = torch.zeros(7, 1, dtype=torch.int32)
    got = routed_experts(layer.hidden.to(DEVICE), gate_up, down, ids.to(DEVICE), gate.to(DEVICE))
    want, bound = plain.layer(layer.hidden, layer.gate_up, layer.down, ids, gate)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("tokens", [1, 24])
def test_replayed_graphs(tokens):
    """Two graphs of the layer over the same weights, replayed in turn with new rows
    and eager work between; every replay equals an eager call, bit for bit."""
    layer = make_layer(hidden=512, width=128, experts=16, top_k=4, rank=16, tokens=tokens, seed=34)
    router = layer.router.to(DEVICE)
    graphs = []
    for fp4 in (False, True):
        gate_up, down = weights_of(layer, fp4)
        x = torch.zeros(tokens, 512, dtype=torch.bfloat16, device=DEVICE)

        def step(x=x, gate_up=gate_up, down=down):
            ids, weights = route(x, router, 4)
            return ids, routed_experts(x, gate_up, down, ids, weights)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, x, step, out))
    g = torch.Generator().manual_seed(9)
    for _ in range(4):
        for graph, x, step, (ids, out) in graphs:
            x.copy_(torch.randn(tokens, 512, generator=g).bfloat16())
            want_ids, want = step()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(ids, want_ids) and torch.equal(out, want)


def test_captured_quantisation():
    g = torch.Generator().manual_seed(10)
    weights = torch.zeros(64, 256, device=DEVICE)
    graph = torch.cuda.CUDAGraph()
    dequantise_fp4(quantise_fp4(weights))
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        values = dequantise_fp4(quantise_fp4(weights))
    for _ in range(3):
        weights.copy_(torch.randn(64, 256, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(values, dequantise_fp4(quantise_fp4(weights)))


def test_two_streams_at_once():
    """Calls on two streams overlap without sharing anything."""
    layer = make_layer(hidden=512, width=256, experts=16, top_k=4, rank=16, tokens=48, seed=35)
    router = layer.router.to(DEVICE)
    gate_up, down = weights_of(layer, False)
    x = [layer.hidden.to(DEVICE), layer.hidden.flip(0).contiguous().to(DEVICE)]
    want = []
    for rows in x:
        ids, weights = route(rows, router, 4)
        want.append(routed_experts(rows, gate_up, down, ids, weights))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = [None, None]
        for n, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                ids, weights = route(x[n], router, 4)
                got[n] = routed_experts(x[n], gate_up, down, ids, weights)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
