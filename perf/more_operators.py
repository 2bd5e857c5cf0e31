"""The operators around a layer's experts, in cases that are timed and compared.

Three kinds of case, each what a user's program runs in one place:

* "rows": tokens laid out by expert and back: the order of a batch's pairs, the
  rows that the experts take and the weighted sum of the rows that they give,
  with `train` also the gradients of both.
* "join": a block's output joined to the residual stream, with the norm behind
  the block, its gate, the residual's scale and the norm before the next block,
  or ("norm") only a norm before a block; with `train` also the gradients.
* "adapters": low-rank adapters of a batch's requests beside one shared
  projection, whose product is given.

`run` computes them in elementary torch operations, or with `own` by the
package's entry points. Hidden sizes, experts and top-k are those of the
benchmark's layers: OLMoE-1B-7B, Qwen3-30B-A3B, a 256-expert layer and Gemma 4.
Hidden states are N(0, 1) with 1 % of the dimensions scaled by 20.
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

EPSILON = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _rows(name: str, tokens: int, hidden: int, experts: int, top_k: int, **options: object) -> dict:
    return {"name": name, "kind": "rows", "tokens": tokens, "hidden": hidden, "experts": experts,
            "top_k": top_k, "type": "bf16", "padded": 0, "absent": 0.0, "zipf": 0.0,
            "ids64": False, "weights16": False, "train": False, **options}


def _join(name: str, tokens: int, hidden: int, **options: object) -> dict:
    return {"name": name, "kind": "join", "tokens": tokens, "hidden": hidden, "type": "bf16",
            "post": False, "next": True, "gate": "none", "scale": 1.0, "weights32": False,
            "train": False, **options}


def _adapters(name: str, tokens: int, hidden: int, outputs: int, adapters: int, rank: int,
              **options: object) -> dict:
    return {"name": name, "kind": "adapters", "tokens": tokens, "hidden": hidden,
            "outputs": outputs, "adapters": adapters, "rank": rank, "bare": 0.0, "runs": False,
            "scaled": True, "ids64": False, **options}


def listed() -> list[dict]:
    return [
        # one stream's token to its eight experts and back: latency is all there is
        _rows("rows-qwen3-t1", 1, 2048, 128, 8),
        # a decode batch padded to its capture size, a quarter of the experts held
        # elsewhere (ids outside the range); int64 ids and BF16 weights
        _rows("rows-gemma4-t122of131", 131, 2816, 128, 8, padded=9, absent=0.25, ids64=True,
              weights16=True),
        # a chunk of prompts through one layer
        _rows("rows-qwen3-t4096", 4096, 2048, 128, 8),
        # a training step's largest batch, skewed routing, forward and backward
        _rows("rows-olmoe-t8191-train", 8191, 2048, 64, 8, zipf=1.2, train=True),
        # FP32 rows of odd sizes, as a check of gradients or a small model trains
        _rows("rows-fp32-t777-train", 777, 1001, 7, 3, type="fp32", train=True),
        # one stream between two blocks: x + block, and the norm of the next block
        _join("join-qwen3-t1", 1, 2048),
        # a decode batch, odd, with a norm behind the block and a residual scale
        _join("join-gemma4-t131", 131, 2816, post=True, scale=0.7, weights32=True),
        # a training step between two blocks, both norms and a gate per channel
        _join("join-olmoe-t8192-train", 8192, 2048, post=True, gate="channel", train=True),
        # FP32 rows of odd sizes with a gate per value
        _join("join-fp32-t515-train", 515, 1003, type="fp32", post=True, gate="full", scale=0.5,
              train=True),
        # one stream with its adapter: latency of reading two small matrices
        _adapters("adapters-qwen3-t1", 1, 2048, 2048, 8, 16),
        # a decode batch in which almost every request has an adapter of its own,
        # beside the gate and up rows of a shared expert
        _adapters("adapters-fine256-t64", 64, 2048, 1024, 64, 32, bare=0.1, ids64=True),
        # prompts of a few requests, one run of tokens each
        _adapters("adapters-prompts-t4001", 4001, 2048, 4096, 5, 64, runs=True),
    ]


def _spread(rng, low: int, high: int) -> int:
    """A whole number of low .. high, even over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    """One more case of the ranges the listed ones stand for."""
    kind = rng.choice(["rows", "join", "norm", "adapters", "adapters"])
    tokens = _spread(rng, 1, 8000)
    if kind == "adapters":
        tokens = min(tokens, 4000)
        return {"kind": kind, "tokens": tokens, "hidden": 8 * rng.randint(32, 256),
                "outputs": 8 * rng.randint(32, 512), "adapters": _spread(rng, 1, 64),
                "rank": 8 * rng.randint(1, 8), "bare": rng.choice([0.0, 0.2]),
                "runs": rng.random() < 0.5, "scaled": rng.random() < 0.7,
                "ids64": rng.random() < 0.5}
    fp32 = rng.random() < 0.3
    hidden = rng.randint(200, 2048) if rng.random() < 0.4 else 128 * rng.randint(2, 16)
    if fp32:
        tokens = min(tokens, 4000)
    case = {"kind": kind, "tokens": tokens, "hidden": hidden, "type": "fp32" if fp32 else "bf16",
            "train": rng.random() < 0.5}
    if kind == "rows":
        experts = _spread(rng, 4, 256)
        return {**case, "experts": experts, "top_k": rng.randint(1, min(8, experts)),
                "padded": rng.randint(1, tokens // 4) if tokens >= 4 and rng.random() < 0.3 else 0,
                "absent": rng.choice([0.0, 0.0, 0.3]), "zipf": rng.choice([0.0, 1.2]),
                "ids64": rng.random() < 0.5, "weights16": rng.random() < 0.5}
    if kind == "norm":
        return {**case, "weights32": rng.random() < 0.5}
    post = rng.random() < 0.5
    return {**case, "post": post, "next": rng.random() < 0.8,
            "gate": rng.choice(["none", "channel", "row", "full"]),
            "scale": rng.choice([1.0, 0.6]), "weights32": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# inputs


def _device() -> torch.device:
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _normal(shape: tuple[int, ...], std: float, g: torch.Generator, dtype: torch.dtype,
            mean: float = 0.0) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=_device()).normal_(mean, std, generator=g)


def _hidden(tokens: int, hidden: int, g: torch.Generator, dtype: torch.dtype) -> torch.Tensor:
    x = torch.randn(tokens, hidden, generator=g, device=_device())
    dims = torch.randperm(hidden, generator=g, device=_device())[: max(1, hidden // 100)]
    x[:, dims] *= 20.0
    return x.to(dtype)


def _routing(case: dict, g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    tokens, experts, device = case["tokens"], case["experts"], _device()
    rank = torch.arange(1, experts + 1, dtype=torch.float64, device=device)
    log_p = -case["zipf"] * torch.log(rank)
    log_p = log_p[torch.randperm(experts, generator=g, device=device)]
    uniform = torch.rand(tokens, experts, generator=g, device=device, dtype=torch.float64)
    top = torch.sort(log_p - torch.log(-torch.log(uniform)), dim=-1, descending=True, stable=True)
    k = case["top_k"]
    ids, weights = top.indices[:, :k], torch.softmax(top.values[:, :k].float(), dim=-1)
    if case["absent"]:
        # experts that another rank holds
        ids = torch.where(ids < experts * (1 - case["absent"]), ids, -1)
    return (ids.to(torch.int64 if case["ids64"] else torch.int32).contiguous(),
            weights.to(torch.bfloat16 if case["weights16"] else torch.float32).contiguous())


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=_device()).manual_seed(seed * 1009 + 2)
    kind, tokens, hidden = case["kind"], case["tokens"], case["hidden"]
    state = {"case": case}
    if kind == "adapters":
        bf16 = torch.bfloat16
        n, rank, outputs = case["adapters"], case["rank"], case["outputs"]
        state["x"] = _hidden(tokens, hidden, g, bf16)
        state["base"] = _normal((tokens, outputs), 1.0, g, bf16)
        state["encoder"] = _normal((n, rank, hidden), hidden ** -0.5, g, bf16)
        state["decoder"] = _normal((n, outputs, rank), 0.05, g, bf16)
        if case["runs"]:
            # each request's tokens in a row; the requests' adapters at random
            ends = torch.sort(torch.randint(0, tokens, (n,), generator=g, device=_device())).values
            request = torch.searchsorted(ends, torch.arange(tokens, device=_device()))
            slots = torch.randperm(n + 1, generator=g, device=_device())[request] % n
        else:
            slots = torch.randint(0, n, (tokens,), generator=g, device=_device())
        bare = torch.rand(tokens, generator=g, device=_device()) < case["bare"]
        slots = torch.where(bare, -1, slots)
        state["slots"] = slots.to(torch.int64 if case["ids64"] else torch.int32)
        state["scales"] = None
        if case["scaled"]:
            state["scales"] = torch.rand(n, generator=g, device=_device()) * 2 + 0.25
        return state
    dtype, train = TYPES[case["type"]], case["train"]
    state["x"] = _hidden(tokens, hidden, g, dtype).requires_grad_(train)
    if kind == "rows":
        ids, weights = _routing(case, g)
        pairs = tokens * case["top_k"]
        state["ids"], state["weights"] = ids, weights.requires_grad_(train)
        state["padding"] = None
        if case["padded"]:
            state["padding"] = torch.arange(tokens, device=_device()) >= tokens - case["padded"]
        # what the experts gave, a row for each pair
        state["rows"] = _normal((pairs, hidden), 0.5, g, dtype).requires_grad_(train)
        if train:
            state["grad_rows"] = _normal((pairs, hidden), 0.01, g, dtype)
            state["grad_out"] = _normal((tokens, hidden), 0.01, g, dtype)
        return state
    weight_type = torch.float32 if case["weights32"] else dtype
    if kind == "norm":
        state["weight"] = _normal((hidden,), 0.1, g, weight_type, 1.0).requires_grad_(train)
        if train:
            state["grad"] = _normal((tokens, hidden), 0.01, g, dtype)
        return state
    state["block"] = _normal((tokens, hidden), 0.5, g, dtype).requires_grad_(train)
    state["post"] = state["next"] = state["gate"] = None
    if case["post"]:
        state["post"] = _normal((hidden,), 0.1, g, weight_type, 1.0).requires_grad_(train)
    if case["next"]:
        state["next"] = _normal((hidden,), 0.1, g, weight_type, 1.0).requires_grad_(train)
    if case["gate"] != "none":
        shape = {"channel": (hidden,), "row": (tokens, 1), "full": (tokens, hidden)}[case["gate"]]
        state["gate"] = _normal(shape, 0.5, g, dtype, 0.5).requires_grad_(train)
    if train:
        state["grad"] = _normal((tokens, hidden), 0.01, g, dtype)
        state["grad_next"] = _normal((tokens, hidden), 0.01, g, dtype) if case["next"] else None
    return state


# ---------------------------------------------------------------------------
# the plain forms


def _plain_rows(s: dict) -> dict:
    case = s["case"]
    experts, k, tokens = case["experts"], case["top_k"], case["tokens"]
    x, products, weights = s["x"].float(), s["rows"].float(), s["weights"].float()
    ids = s["ids"]
    kept = (ids >= 0) & (ids < experts)
    if s["padding"] is not None:
        kept = kept & ~s["padding"].unsqueeze(-1)
    key = torch.where(kept, ids, experts).flatten()
    ranked, pairs = torch.sort(key, stable=True)
    row = torch.empty_like(pairs)
    row[pairs] = torch.arange(pairs.numel(), device=pairs.device)
    row = row.view(tokens, k)
    offsets = torch.searchsorted(ranked, torch.arange(experts + 1, device=key.device, dtype=key.dtype))
    live = (ranked < experts).unsqueeze(-1)
    dtype = s["x"].dtype
    result = {"offsets": offsets.int(), "places": torch.where(kept, row, -1 - row).int(),
              "pairs": pairs.int(),
              "rows": torch.where(live, x[pairs // k], 0.0).to(dtype)}
    mixed = products[row] * weights.unsqueeze(-1)
    result["out"] = torch.where(kept.unsqueeze(-1), mixed, 0.0).sum(1).to(dtype)
    if case["train"]:
        back, grad_out = s["grad_rows"].float()[row], s["grad_out"].float()
        result["x"] = torch.where(kept.unsqueeze(-1), back, 0.0).sum(1).to(dtype)
        result["products"] = torch.where(
            live, grad_out[pairs // k] * weights.flatten()[pairs].unsqueeze(-1), 0.0).to(dtype)
        dots = (products[row] * grad_out.unsqueeze(1)).sum(-1)
        result["weights"] = torch.where(kept, dots, 0.0).to(s["weights"].dtype)
    return result


def _unit(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(x over the root of its mean square, one over that root)."""
    inverse = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON)
    return x * inverse, inverse


def _unit_back(grad: torch.Tensor, unit: torch.Tensor, inverse: torch.Tensor) -> torch.Tensor:
    return inverse * (grad - unit * (grad * unit).mean(-1, keepdim=True))


def _plain_norm(s: dict) -> dict:
    dtype, weight = s["x"].dtype, s["weight"].float()
    unit, inverse = _unit(s["x"].float())
    result = {"out": (unit * weight).to(dtype)}
    if s["case"]["train"]:
        grad = s["grad"].float()
        result["x"] = _unit_back(grad * weight, unit, inverse).to(dtype)
        result["weight"] = (grad * unit).sum(0).to(s["weight"].dtype)
    return result


def _plain_join(s: dict) -> dict:
    case, dtype = s["case"], s["x"].dtype
    block = s["block"].float()
    inner = block
    if s["post"] is not None:
        block_unit, block_inverse = _unit(block)
        inner = block_unit * s["post"].float()
    gated = inner if s["gate"] is None else inner * s["gate"].float()
    joined = case["scale"] * s["x"].float() + gated
    result = {"joined": joined.to(dtype)}
    if s["next"] is not None:
        unit, inverse = _unit(joined)
        result["out"] = (unit * s["next"].float()).to(dtype)
    if not case["train"]:
        return result
    grad = s["grad"].float()
    if s["next"] is not None:
        grad_next = s["grad_next"].float()
        grad = grad + _unit_back(grad_next * s["next"].float(), unit, inverse)
        result["next"] = (grad_next * unit).sum(0).to(s["next"].dtype)
    result["x"] = (case["scale"] * grad).to(dtype)
    inner_grad = grad
    if s["gate"] is not None:
        inner_grad = grad * s["gate"].float()
        both = grad * inner
        if case["gate"] == "channel":
            both = both.sum(0)
        elif case["gate"] == "row":
            both = both.sum(-1, keepdim=True)
        result["gate"] = both.to(s["gate"].dtype)
    if s["post"] is not None:
        result["post"] = (inner_grad * block_unit).sum(0).to(s["post"].dtype)
        inner_grad = _unit_back(inner_grad * s["post"].float(), block_unit, block_inverse)
    result["block"] = inner_grad.to(dtype)
    return result


def _plain_adapters(s: dict) -> dict:
    case = s["case"]
    n, rank, tokens = case["adapters"], case["rank"], case["tokens"]
    x, base, slots = s["x"].float(), s["base"].float(), s["slots"].long()
    kept = (slots >= 0) & (slots < n)
    slot = torch.where(kept, slots, 0)
    scale = kept.float() if s["scales"] is None else torch.where(kept, s["scales"][slot], 0.0)
    if tokens <= 4 * n:  # few tokens: each one's adapter
        inner = torch.matmul(s["encoder"][slot].float(), x.unsqueeze(-1))
        delta = torch.matmul(s["decoder"][slot].float(), inner).squeeze(-1) * scale.unsqueeze(-1)
    else:  # many: every adapter's inner values, all but the token's own cleared
        inner = torch.matmul(x, s["encoder"].float().flatten(0, 1).T).view(tokens, n, rank)
        chosen = slot.unsqueeze(-1) == torch.arange(n, device=x.device)
        inner = torch.where(chosen.unsqueeze(-1), inner * scale[:, None, None], 0.0)
        delta = torch.matmul(inner.view(tokens, n * rank),
                             s["decoder"].float().transpose(1, 2).reshape(n * rank, -1))
    return {"out": (base + delta).bfloat16()}


def run(state: dict) -> dict:
    kind = state["case"]["kind"]
    if own:
        return _own(state)
    with torch.no_grad():
        return {"rows": _plain_rows, "norm": _plain_norm, "join": _plain_join,
                "adapters": _plain_adapters}[kind](state)


# ---------------------------------------------------------------------------
# the package's entry points


def _own(s: dict) -> dict:
    case, kind = s["case"], s["case"]["kind"]
    if kind == "adapters":
        from calibration_free_moe.reader.adapters import apply_adapters

        return {"out": apply_adapters(s["base"], s["x"], s["encoder"], s["decoder"], s["slots"],
                                      s["scales"])}
    if kind == "rows":
        from calibration_free_moe.reader.dispatch import combine_rows, gather_rows, sort_by_expert

        order = sort_by_expert(s["ids"], case["experts"], s["padding"])
        rows = gather_rows(s["x"], order)
        out = combine_rows(s["rows"], order, s["weights"])
        result = {"offsets": order.offsets, "places": order.places, "pairs": order.pairs,
                  "rows": rows.detach(), "out": out.detach()}
        if case["train"]:
            result["x"], result["products"], result["weights"] = torch.autograd.grad(
                (rows, out), (s["x"], s["rows"], s["weights"]), (s["grad_rows"], s["grad_out"]))
        return result
    from calibration_free_moe.reader.norms import join_block, norm_rows

    if kind == "norm":
        out = norm_rows(s["x"], s["weight"], epsilon=EPSILON)
        result = {"out": out.detach()}
        if case["train"]:
            result["x"], result["weight"] = torch.autograd.grad(
                out, (s["x"], s["weight"]), s["grad"])
        return result
    joined = join_block(s["x"], s["block"], post_weight=s["post"], gate=s["gate"],
                        residual_scale=case["scale"], next_weight=s["next"], epsilon=EPSILON)
    outputs, grads = (joined,), (s.get("grad"),)
    if s["next"] is not None:
        outputs, grads = joined, (s.get("grad"), s.get("grad_next"))
    result = dict(zip(("joined", "out"), (o.detach() for o in outputs)))
    if case["train"]:
        leaves = {name: s[name] for name in ("x", "block", "post", "next", "gate")
                  if s[name] is not None}
        result.update(zip(leaves, torch.autograd.grad(outputs, tuple(leaves.values()), grads)))
    return result


# ---------------------------------------------------------------------------
# work, and the same in 64 bits


def work(case: dict) -> dict:
    kind, tokens, hidden = case["kind"], case["tokens"], case["hidden"]
    if kind == "adapters":
        n, rank, outputs = case["adapters"], case["rank"], case["outputs"]
        live = tokens * (1 - case["bare"])
        touched = min(n, live) if case["runs"] else n * (1 - (1 - 1 / n) ** live)
        return {"bytes": 2 * (live * hidden + 2 * tokens * outputs
                              + touched * rank * (hidden + outputs))
                + tokens * (8 if case["ids64"] else 4),
                "flops": 2 * live * rank * (hidden + outputs)}
    size = 4 if case["type"] == "fp32" else 2
    row = tokens * hidden * size
    if kind == "rows":
        k = case["top_k"]
        live = k * (1 - case["padded"] / tokens) * (1 - case["absent"])
        ids = tokens * k * ((8 if case["ids64"] else 4) + 8)
        weights = tokens * k * (2 if case["weights16"] else 4)
        # rows in, a row for each pair out; those that the experts gave in, the sum out
        bytes_, flops = ids + weights + row * (1 + k) + row * (live + 1), 2 * live * tokens * hidden
        if case["train"]:
            # of the rows: one for each pair in, the sum out; of the sum: its gradient and
            # the experts' rows in, a row for each pair out
            bytes_ += 2 * weights + row * (live + 1) + row * (1 + live + k)
            flops += 4 * live * tokens * hidden
        return {"bytes": bytes_, "flops": flops}
    if kind == "norm":
        return {"bytes": row * (5 if case["train"] else 2),
                "flops": tokens * hidden * (14 if case["train"] else 4)}
    gate = {"none": 0, "channel": 0, "row": 0, "full": row}[case["gate"]]
    outputs = 2 if case["next"] else 1
    flops = 2 + 4 * case["post"] + 4 * case["next"] + (case["gate"] != "none")
    total = 2 * row + gate + outputs * row
    if case["train"]:
        total += outputs * row + 2 * row + gate + 2 * row + gate
        flops *= 3
    return {"bytes": total, "flops": flops * tokens * hidden}


def _exact_unit(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    root = torch.sqrt(torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / x.shape[1] + EPSILON)
    return x / root, root


def _exact_unit_back(x: torch.Tensor, root: torch.Tensor, grad: torch.Tensor) -> torch.Tensor:
    along = (grad * x).sum(1, keepdim=True) / x.shape[1]
    return grad / root - x * along / root ** 3


def _exact_rows(s: dict) -> dict:
    """Expert after expert, each one's pairs in the batch's order."""
    case = s["case"]
    experts, k, tokens, hidden = case["experts"], case["top_k"], case["tokens"], case["hidden"]
    x, products, weights = s["x"].double(), s["rows"].double(), s["weights"].double()
    ids = s["ids"].clone()
    ids[(ids < 0) | (ids >= experts)] = experts
    if s["padding"] is not None:
        ids[s["padding"]] = experts
    pairs = torch.cat([torch.nonzero(ids.flatten() == e).flatten() for e in range(experts + 1)])
    counts = [int((ids == e).sum()) for e in range(experts)]
    starts = [sum(counts[:e]) for e in range(experts + 1)]
    count = starts[-1]
    token, slot = pairs[:count] // k, pairs[:count] % k
    places = torch.empty(tokens, k, dtype=torch.int64, device=x.device)
    place = torch.arange(tokens * k, device=x.device)
    places[pairs // k, pairs % k] = torch.where(place < count, place, -1 - place)
    rows = torch.zeros(tokens * k, hidden, dtype=torch.float64, device=x.device)
    rows[:count] = x[token]
    out = torch.zeros_like(x)
    out.index_add_(0, token, products[:count] * weights[token, slot].unsqueeze(-1))
    result = {"offsets": torch.tensor(starts, device=x.device), "places": places, "pairs": pairs,
              "rows": rows, "out": out}
    if case["train"]:
        grad_rows, grad_out = s["grad_rows"].double(), s["grad_out"].double()
        result["x"] = torch.zeros_like(x).index_add_(0, token, grad_rows[:count])
        result["products"] = torch.zeros_like(rows)
        result["products"][:count] = grad_out[token] * weights[token, slot].unsqueeze(-1)
        result["weights"] = torch.zeros_like(weights)
        result["weights"][token, slot] = torch.linalg.vecdot(grad_out[token], products[:count])
    return result


def exact(case: dict, seed: int) -> dict:
    s = {name: v.detach() if isinstance(v, torch.Tensor) else v
         for name, v in prepare(case, seed).items()}
    kind, x = case["kind"], s["x"].double()
    if kind == "rows":
        return _exact_rows(s)
    if kind == "norm":
        unit, root = _exact_unit(x)
        weight = s["weight"].double()
        result = {"out": unit * weight}
        if case["train"]:
            grad = s["grad"].double()
            result["x"] = _exact_unit_back(x, root, grad * weight)
            result["weight"] = (grad * unit).sum(dim=0)
        return result
    if kind == "adapters":
        out = s["base"].double()
        for a in range(case["adapters"]):
            token = torch.nonzero(s["slots"] == a).flatten()
            both = s["decoder"][a].double() @ (s["encoder"][a].double() @ x[token].T)
            out[token] += both.T * (1.0 if s["scales"] is None else s["scales"][a].double())
        return {"out": out}
    block, ones = s["block"].double(), torch.ones_like(x)
    gate = ones if s["gate"] is None else s["gate"].double().expand_as(x)
    post = ones if s["post"] is None else s["post"].double().expand_as(x)
    unit, root = (block, ones) if s["post"] is None else _exact_unit(block)
    joined = case["scale"] * x + gate * post * unit
    result = {"joined": joined}
    if s["next"] is not None:
        next_unit, next_root = _exact_unit(joined)
        result["out"] = next_unit * s["next"].double()
    if not case["train"]:
        return result
    grad = s["grad"].double()
    if s["next"] is not None:
        grad_next = s["grad_next"].double()
        result["next"] = (grad_next * next_unit).sum(dim=0)
        grad = grad + _exact_unit_back(joined, next_root, grad_next * s["next"].double())
    result["x"] = grad * case["scale"]
    if s["gate"] is not None:
        result["gate"] = (grad * post * unit).sum_to_size(s["gate"].shape)
    if s["post"] is not None:
        result["post"] = (grad * gate * unit).sum(dim=0)
        result["block"] = _exact_unit_back(block, root, grad * gate * post)
    else:
        result["block"] = grad * gate
    return result
