"""The operators beside the sparse reader, in cases that are timed and compared.

Three kinds of case, each one call (or a pair of calls) of a user's program:

* "route": the router of one layer, hidden rows to expert ids and weights.
* "experts": one mixture-of-experts layer read whole, over BF16 weights or over
  microscaled 4-bit ones (`format`).
* "quantise": weights to microscaled 4-bit floating point and back to values.

`run` computes them in elementary torch operations, or with `own` by the
package's entry points. Shapes are those of the benchmark's layers:
OLMoE-1B-7B, Qwen3-30B-A3B, a 256-expert layer and Gemma 4. Weights are
N(0, 0.02^2), hidden states N(0, 1) with 1 % of the dimensions scaled by 20;
experts come from a softmax router, or from a Zipf popularity law by Gumbel
top-k.
"""

from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(
    0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "calibration-free-moe_amd")
)

own = False

# hidden, width, experts, top-k, activation
SHAPES = {
    "olmoe": (2048, 1024, 64, 8, "silu"),
    "qwen3": (2048, 768, 128, 8, "silu"),
    "fine256": (2048, 512, 256, 8, "silu"),
    "gemma4": (2816, 704, 128, 8, "gelu_tanh"),
}

BLOCK = 32  # values that share a scale


def _layer(shape: str) -> dict:
    hidden, width, experts, top_k, activation = SHAPES[shape]
    return {"hidden": hidden, "width": width, "experts": experts, "top_k": top_k,
            "activation": activation}


def _route(name: str, shape: str, tokens: int, **options: object) -> dict:
    layer = _layer(shape)
    return {"name": name, "kind": "route", "hidden": layer["hidden"], "experts": layer["experts"],
            "top_k": layer["top_k"], "tokens": tokens, "renormalise": True, "scaled": False,
            "ids64": False, "weights16": False, **options}


def _experts(name: str, shape: str, tokens: int, **options: object) -> dict:
    return {"name": name, "kind": "experts", "format": "bf16", **_layer(shape), "tokens": tokens,
            "padded": 0, "zipf": 0.0, "ids64": False, "weights16": False, **options}


def listed() -> list[dict]:
    return [
        # one stream's router: latency is all there is
        _route("route-qwen3-t1", "qwen3", 1),
        # a full decode batch, odd, with a scale per expert and BF16 weights and
        # int64 ids, as Gemma 4's router gives them
        _route("route-gemma4-t131", "gemma4", 131, scaled=True, ids64=True, weights16=True),
        # a chunk of prompts through the fine-grained layer's router, ragged;
        # weights of the whole softmax, not renormalised
        _route("route-fine256-t4001", "fine256", 4001, renormalise=False),
        # single-stream decoding: one token through one layer
        _experts("experts-qwen3-t1", "qwen3", 1),
        # a small batch padded to its capture size; hidden size 2816, GELU
        _experts("experts-gemma4-t13of16", "gemma4", 16, padded=3, ids64=True, weights16=True),
        # the benchmark's headline batch, every expert touched
        _experts("experts-olmoe-t64", "olmoe", 64),
        # the largest batch, skewed routing: some experts get a hundred tokens
        _experts("experts-qwen3-t256-zipf", "qwen3", 256, zipf=1.2),
        # single-stream decoding from 4-bit experts: latency of the launches
        _experts("experts4-qwen3-t1", "qwen3", 1, format="fp4"),
        # a handful of streams on the fine-grained layer
        _experts("experts4-fine256-t5", "fine256", 5, format="fp4", ids64=True),
        # a full decode batch over 4-bit experts
        _experts("experts4-qwen3-t128", "qwen3", 128, format="fp4"),
        # a shared expert's gate/up rows from FP32 master weights
        {"name": "quantise-shared", "kind": "quantise", "rows": 1024, "columns": 2048,
         "master": True},
        # model loading: the gate/up rows of a whole layer
        {"name": "quantise-qwen3-layer", "kind": "quantise", "rows": 128 * 1536, "columns": 2048,
         "master": False},
    ]


def _spread(rng, low: int, high: int) -> int:
    """A whole number of low .. high, even over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    """One more case of the ranges the listed ones stand for."""
    kind = rng.choice(["route", "experts", "experts", "experts4", "experts4", "quantise"])
    if kind == "quantise":
        columns = BLOCK * rng.randint(4, 128)
        return {"kind": "quantise", "rows": _spread(rng, 200, 300_000_000 // columns),
                "columns": columns, "master": rng.random() < 0.3}
    if kind == "route":
        experts = rng.randint(8, 256)
        return {"kind": "route", "hidden": 128 * rng.randint(4, 16), "experts": experts,
                "top_k": rng.randint(1, min(10, experts)), "tokens": _spread(rng, 1, 4000),
                "renormalise": rng.random() < 0.5, "scaled": rng.random() < 0.3,
                "ids64": rng.random() < 0.5, "weights16": rng.random() < 0.5}
    fp4 = kind == "experts4"
    hidden = 128 * rng.randint(4, 24)
    width = 32 * rng.randint(4, 32) if fp4 else 16 * rng.randint(8, 64)
    most = min(200, 600_000_000 // (3 * width * hidden))
    experts = _spread(rng, min(8, most), most)
    tokens = _spread(rng, 1, 250)
    return {"kind": "experts", "format": "fp4" if fp4 else "bf16", "hidden": hidden,
            "width": width, "experts": experts, "top_k": rng.randint(1, min(8, experts)),
            "activation": rng.choice(["silu", "silu", "gelu_tanh"]), "tokens": tokens,
            "padded": rng.randint(1, tokens // 4) if tokens >= 4 and rng.random() < 0.3 else 0,
            "zipf": rng.choice([0.0, 0.0, 1.2]), "ids64": rng.random() < 0.5,
            "weights16": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# inputs


def _device() -> torch.device:
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _normal(shape: tuple[int, ...], std: float, g: torch.Generator,
            dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=_device()).normal_(0.0, std, generator=g)


def _hidden(tokens: int, hidden: int, g: torch.Generator) -> torch.Tensor:
    x = torch.randn(tokens, hidden, generator=g, device=_device())
    dims = torch.randperm(hidden, generator=g, device=_device())[: max(1, hidden // 100)]
    x[:, dims] *= 20.0
    return x.bfloat16()


def _routing(case: dict, x: torch.Tensor, g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    experts, device = case["experts"], _device()
    if case["zipf"]:
        rank = torch.arange(1, experts + 1, dtype=torch.float64, device=device)
        log_p = -case["zipf"] * torch.log(rank)
        log_p = log_p[torch.randperm(experts, generator=g, device=device)]
        uniform = torch.rand(x.shape[0], experts, generator=g, device=device, dtype=torch.float64)
        logits = log_p - torch.log(-torch.log(uniform))
    else:
        logits = x.float() @ _normal((experts, case["hidden"]), 0.02, g).float().T
    top = torch.sort(logits, dim=-1, descending=True, stable=True)
    k = case["top_k"]
    ids, weights = top.indices[:, :k], torch.softmax(top.values[:, :k], dim=-1)
    return (ids.to(torch.int64 if case["ids64"] else torch.int32).contiguous(),
            weights.to(torch.bfloat16 if case["weights16"] else torch.float32).contiguous())


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=_device()).manual_seed(seed * 1009 + 1)
    if case["kind"] == "quantise":
        dtype = torch.float32 if case["master"] else torch.bfloat16
        return {"case": case, "weights": _normal((case["rows"], case["columns"]), 0.02, g, dtype)}
    x = _hidden(case["tokens"], case["hidden"], g)
    if case["kind"] == "route":
        scale = None
        if case["scaled"]:
            scale = torch.rand(case["experts"], generator=g, device=_device()) + 0.5
        return {"case": case, "x": x, "scale": scale,
                "router": _normal((case["experts"], case["hidden"]), 0.02, g)}
    ids, weights = _routing(case, x, g)
    experts, width, hidden = case["experts"], case["width"], case["hidden"]
    gate_up = _normal((experts, 2 * width, hidden), 0.02, g)
    padding = None
    if case["padded"]:
        padding = torch.arange(case["tokens"], device=_device()) >= case["tokens"] - case["padded"]
    if case["format"] == "fp4":
        # codes and scales as a checkpoint holds them
        gate_up = _plain_quantise(gate_up)
        down = _plain_quantise(_normal((experts, hidden, width), 0.02, g))
    else:
        # channel-major, as the reader borrows it
        down = _normal((experts, width, hidden), 0.02, g).transpose(1, 2)
    return {"case": case, "x": x, "gate_up": gate_up, "down": down, "ids": ids,
            "weights": weights, "padding": padding}


# ---------------------------------------------------------------------------
# the plain forms


def _plain_quantise(weights: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales): two E2M1 codes a byte, the even element low; E8M0 bytes."""
    value = weights.float().unflatten(-1, (-1, BLOCK))
    largest = value.abs().amax(-1)
    exponent = torch.frexp(largest).exponent - 1
    byte = torch.where(largest > 0, exponent + 125, 0).clamp(2, 254)
    byte = torch.where(torch.isfinite(largest), byte, 255).to(torch.int32)
    inverse = ((254 - byte.clamp(max=252)) << 23).view(torch.float32)
    scaled = (value * inverse.unsqueeze(-1)).abs()
    fine = torch.round(2 * scaled)  # (to even, as everywhere below)
    code = torch.where(scaled < 2, fine, torch.where(scaled < 4, torch.round(scaled) + 2,
                                                     torch.round(scaled / 2) + 4))
    code = code.clamp(max=7).to(torch.uint8) | (torch.signbit(value).to(torch.uint8) << 3)
    code = torch.where((byte == 255).unsqueeze(-1), 0, code).to(torch.uint8).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _plain_values(fp4: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
    """The FP32 values that codes and scales stand for."""
    codes, scales = fp4
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat([table, -table])
    value = table[torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).int()]
    scale = (scales.to(torch.int32) << 23).view(torch.float32)
    scale = torch.where(scales == 255, math.nan, scale)
    scale = torch.where(scales == 0, 2.0 ** -127, scale)
    return (value.unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)


def _plain_route(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    case, k = s["case"], s["case"]["top_k"]
    # (64 bits: neighbours about the cut may differ by less than an FP32 sum is off)
    logits = s["x"].double() @ s["router"].double().T
    top = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids = top.indices[:, :k]
    share = torch.exp((top.values - top.values[:, :1]).float())
    total = share[:, :k] if case["renormalise"] else share
    weights = share[:, :k] / total.sum(-1, keepdim=True)
    if s["scale"] is not None:
        weights = weights * s["scale"][ids]
    return (ids.to(torch.int64 if case["ids64"] else torch.int32),
            weights.to(torch.bfloat16 if case["weights16"] else torch.float32))


def _phi(gate: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "silu":
        return gate / (1 + torch.exp(-gate))
    inner = math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate)
    return 0.5 * gate * (1 + torch.tanh(inner))


def _plain_experts(s: dict) -> torch.Tensor:
    case, width = s["case"], s["case"]["width"]
    fp4 = case["format"] == "fp4"
    x, ids, weights = s["x"].float(), s["ids"].long(), s["weights"].float()
    tokens, experts = case["tokens"], case["experts"]
    if ids.numel() <= experts:  # few pairs: each one's expert
        if fp4:
            gate_up = _plain_values([v[ids] for v in s["gate_up"]])
            down = _plain_values([v[ids] for v in s["down"]])
        else:
            gate_up, down = s["gate_up"][ids].float(), s["down"][ids].float()
        both = torch.matmul(gate_up, x[:, None, :, None]).squeeze(-1)
        act = _phi(both[..., :width], case["activation"]) * both[..., width:]
        out = (torch.matmul(down, act.unsqueeze(-1)).squeeze(-1) * weights.unsqueeze(-1)).sum(1)
    else:  # many: every expert's output for every token, mixed by its weight
        gate_up = _plain_values(s["gate_up"]) if fp4 else s["gate_up"].float()
        down = _plain_values(s["down"]) if fp4 else s["down"].float()
        mix = torch.zeros(tokens, experts, device=x.device).scatter_add_(1, ids, weights)
        both = torch.matmul(x, gate_up.transpose(1, 2))
        act = _phi(both[..., :width], case["activation"]) * both[..., width:]
        out = torch.matmul(act * mix.T.unsqueeze(-1), down.transpose(1, 2)).sum(0)
    if s["padding"] is not None:
        out = torch.where(s["padding"].unsqueeze(-1), 0.0, out)
    return out.bfloat16()


def run(state: dict) -> dict:
    kind = state["case"]["kind"]
    if own:
        return _own(state)
    if kind == "route":
        ids, weights = _plain_route(state)
        return {"ids": ids, "weights": weights}
    if kind == "experts":
        return {"out": _plain_experts(state)}
    return {"values": _plain_values(_plain_quantise(state["weights"])).bfloat16()}


# ---------------------------------------------------------------------------
# the package's entry points


def _own(s: dict) -> dict:
    case = s["case"]
    if case["kind"] == "route":
        from calibration_free_moe.reader.router import route

        ids, weights = route(
            s["x"], s["router"], case["top_k"], renormalise=case["renormalise"],
            expert_scale=s["scale"], ids_dtype=torch.int64 if case["ids64"] else torch.int32,
            weights_dtype=torch.bfloat16 if case["weights16"] else torch.float32)
        return {"ids": ids, "weights": weights}
    from calibration_free_moe.reader.microscale import Fp4Weights, dequantise_fp4, quantise_fp4

    if case["kind"] == "quantise":
        return {"values": dequantise_fp4(quantise_fp4(s["weights"]))}
    from calibration_free_moe.reader.experts import routed_experts

    gate_up, down = s["gate_up"], s["down"]
    if case["format"] == "fp4":
        gate_up, down = Fp4Weights(*gate_up), Fp4Weights(*down)
    return {"out": routed_experts(s["x"], gate_up, down, s["ids"], s["weights"], s["padding"],
                                  activation=case["activation"])}


# ---------------------------------------------------------------------------
# work, and the same in 64 bits


def _touched(case: dict) -> float:
    """Expected number of experts that some token of the batch is sent to."""
    experts, top_k = case["experts"], case["top_k"]
    tokens = case["tokens"] - case["padded"]
    if not case["zipf"]:
        return experts * (1 - (1 - top_k / experts) ** tokens)
    p = [(r + 1) ** -case["zipf"] for r in range(experts)]
    total = sum(p)
    low, high = 1.0, 1e6  # draws that give top_k different experts a token
    for _ in range(60):
        m = math.sqrt(low * high)
        low, high = (m, high) if sum(1 - (1 - v / total) ** m for v in p) < top_k else (low, m)
    return sum(1 - (1 - v / total) ** (low * tokens) for v in p)


def work(case: dict) -> dict:
    if case["kind"] == "quantise":
        # weights in, codes and scales out, values out; about ten operations a value
        values = case["rows"] * case["columns"]
        held = values * (1 / 2 + 1 / BLOCK)
        return {"bytes": (4 if case["master"] else 2) * values + held + 2 * values,
                "flops": 10 * values}
    hidden, experts, tokens = case["hidden"], case["experts"], case["tokens"]
    routed = tokens * case["top_k"] * ((8 if case["ids64"] else 4) + (2 if case["weights16"] else 4))
    if case["kind"] == "route":
        return {"bytes": 2 * hidden * (tokens + experts) + routed,
                "flops": 2 * tokens * experts * hidden}
    bytes_each = 2 if case["format"] == "bf16" else 1 / 2 + 1 / BLOCK
    live = tokens - case["padded"]
    return {"bytes": _touched(case) * 3 * case["width"] * hidden * bytes_each
            + 2 * hidden * (live + tokens) + routed,
            "flops": 6 * live * case["top_k"] * case["width"] * hidden}


def _exact_values(weights: torch.Tensor) -> torch.Tensor:
    """Quantised and back, by counting the borders of the grid below each value."""
    value = weights.double().reshape(weights.shape[0], -1, BLOCK)
    largest = value.abs().max(-1, keepdim=True).values
    scale = torch.exp2(torch.floor(torch.log2(largest.clamp_min(2.0 ** -123))) - 2)
    scaled = value.abs() / scale
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=value.device)
    place = (scaled > 0.25).int()
    for border, even in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True),
                         (5.0, False)):
        # a tie goes to the neighbour whose last mantissa bit is zero
        place += (scaled >= border) if even else (scaled > border)
    return (grid[place] * scale * torch.sign(value)).reshape(weights.shape)


def _exact_unpack(fp4: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
    codes, scales = fp4
    nibble = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.int64,
                         device=codes.device)
    nibble[..., 0::2] = (codes % 16).long()
    nibble[..., 1::2] = (codes // 16).long()
    magnitude, sign = nibble % 8, 1.0 - 2.0 * (nibble // 8).double()
    power, half = magnitude // 2, (magnitude % 2).double()
    value = torch.where(power == 0, half / 2, torch.exp2(power.double() - 1) * (1 + half / 2))
    scale = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=-1)
    return sign * value * scale


def exact(case: dict, seed: int) -> dict:
    s = prepare(case, seed)
    if case["kind"] == "quantise":
        # (in pieces: the 64-bit forms of a whole layer are large)
        return {"values": torch.cat([_exact_values(part) for part in s["weights"].split(16384)])}
    if case["kind"] == "route":
        logits = torch.matmul(s["router"].double(), s["x"].double().T).T
        order = torch.argsort(-logits, dim=-1, stable=True)[:, : case["top_k"]]
        chosen = torch.gather(logits, 1, order)
        base = chosen if case["renormalise"] else logits
        weights = torch.exp(chosen - torch.logsumexp(base, dim=-1, keepdim=True))
        if s["scale"] is not None:
            weights = weights * s["scale"].double()[order]
        return {"ids": order, "weights": weights}
    width = case["width"]
    out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=s["x"].device)
    for expert in range(case["experts"]):
        token, slot = torch.nonzero(s["ids"] == expert, as_tuple=True)
        if not token.numel():
            continue
        if case["format"] == "fp4":
            gate_up = _exact_unpack([v[expert] for v in s["gate_up"]])
            down = _exact_unpack([v[expert] for v in s["down"]])
        else:
            gate_up, down = s["gate_up"][expert].double(), s["down"][expert].double()
        both = s["x"][token].double() @ gate_up.T
        gate, up = both[:, :width], both[:, width:]
        if case["activation"] == "silu":
            act = gate * torch.sigmoid(gate) * up
        else:
            cubic = gate + 0.044715 * gate ** 3
            act = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * cubic)) * up
        part = (act @ down.T) * s["weights"][token, slot].double().unsqueeze(-1)
        out.index_add_(0, token, part)
    if s["padding"] is not None:
        out[s["padding"]] = 0.0
    return {"out": out}
