"""Microscaled 4-bit floating point, as cases to time and to compare: the quantisation of rows, products of quantised rows with such
weights, a feed-forward's gated unit between two of them, and routed experts.

A row is cut into blocks of 32 values that share a power of two: with e = floor(log2(largest magnitude)) - 2, at least -127, a value is
2^e times one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 or its negative: the nearest to it, ties to the even code, 6 where it is larger. What a product takes on its
left is quantised on the way, a weight when a model is loaded; sums are exact products of such values. A gated unit's result is
quantised as it is, without a rounding in between.

A case is a dict of plain values. With ``own`` the framework's calls are made, else the plain forms below.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
BLOCK = 32
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bfloat16": BF16, "float32": F32}
STEPS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one request's token before a projection: launches and latency
        dict(name="quantise_1x5120", op="quantise", tokens=1, k=5120, experts=0, top_k=1, dtype="bfloat16"),
        # a long prompt's activations, unrounded: what moves is what counts
        dict(name="quantise_8001x8192_f32", op="quantise", tokens=8001, k=8192, experts=0, top_k=1, dtype="float32"),
        # a prompt's rows on their way to the experts, two a token
        dict(name="quantise_1987x5120_sorted", op="quantise", tokens=1987, k=5120, experts=16, top_k=2, dtype="bfloat16"),
        # one token through a small projection
        dict(name="linear_1x2048x2048", op="linear", tokens=1, n_out=2048, k=2048, bias=False, out="bfloat16"),
        # eight requests' tokens through q, k and v, with a bias
        dict(name="linear_8x7168x5120", op="linear", tokens=8, n_out=7168, k=5120, bias=True, out="bfloat16"),
        # a step of many requests and a short portion: an odd number of tokens, unrounded sums
        dict(name="linear_99x5120x8192_f32", op="linear", tokens=99, n_out=5120, k=8192, bias=False, out="float32"),
        # a prompt through a wide projection
        dict(name="linear_2048x16384x5120", op="linear", tokens=2048, n_out=16384, k=5120, bias=False, out="bfloat16"),
        # one token through a dense feed-forward: the weights are what moves
        dict(name="feed_forward_1x5120x8192", op="feed_forward", tokens=1, hidden=5120, inter=8192, limit=0.0),
        # a prompt through it, an odd number of tokens, the clamped unit
        dict(name="feed_forward_2047x5120x8192", op="feed_forward", tokens=2047, hidden=5120, inter=8192, limit=7.0),
        # eight requests' tokens through routed experts, the score on what an expert reads
        dict(name="experts_8_1of16", op="experts", tokens=8, hidden=5120, inter=8192, experts=16, top_k=1, scale="input",
             limit=0.0),
        # a full serving batch through many narrow experts, the score on what they return
        dict(name="experts_64_6of64", op="experts", tokens=64, hidden=2048, inter=1024, experts=64, top_k=6, scale="output",
             limit=0.0),
        # a prompt through the wide ones
        dict(name="experts_2048_1of16", op="experts", tokens=2048, hidden=5120, inter=8192, experts=16, top_k=1, scale="input",
             limit=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["quantise", "linear", "linear", "feed_forward", "experts"])
    blocks = lambda lo, hi: BLOCK * max(1, round(_log(rng, lo, hi) / BLOCK))
    if op == "quantise":
        experts = rng.choice([0, 0, 8, 16, 64])
        return dict(op=op, tokens=_log(rng, 1, 4000), k=blocks(256, 8192), experts=experts,
                    top_k=rng.choice([1, 2, 4]) if experts else 1, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    tokens = _log(rng, 1, 2048)
    if op == "linear":
        return dict(op=op, tokens=tokens, n_out=_log(rng, 64, 16384), k=blocks(256, 5120), bias=rng.random() < 0.3,
                    out=rng.choice(["bfloat16", "bfloat16", "float32"]))
    limit = rng.choice([0.0, 0.0, 7.0])
    if op == "feed_forward":
        return dict(op=op, tokens=tokens, hidden=blocks(256, 5120), inter=blocks(256, 8192), limit=limit)
    experts = rng.choice([4, 8, 16, 64])
    top_k = rng.choice([1, 1, 2, 4])
    most = 16 * 5120 * 8192 // experts                              # of one expert's stacks
    hidden = blocks(256, 5120)
    inter = BLOCK * max(1, min(blocks(256, 8192), most // hidden) // BLOCK)
    return dict(op=op, tokens=max(1, tokens // top_k), hidden=hidden, inter=inter, experts=experts, top_k=top_k,
                scale=rng.choice(["input", "output"]) if limit == 0.0 else "output", limit=limit)


def _held(rows, k):
    """Bytes of rows of k values: half a byte each, and one for every block."""
    return rows * (k // 2 + k // BLOCK)


def work(case):
    n = case["tokens"]
    if case["op"] == "quantise":
        k, rows = case["k"], n * case["top_k"]
        read = n * k * (4 if case["dtype"] == "float32" else 2)
        return {"bytes": read + 2 * _held(rows, k) + 2 * rows * k, "flops": 4 * rows * k}
    if case["op"] == "linear":
        m, k = case["n_out"], case["k"]
        out = n * m * (4 if case["out"] == "float32" else 2)
        return {"bytes": _held(m, k) + 2 * n * k + out + (2 * m if case["bias"] else 0), "flops": 2 * n * m * k}
    h, i = case["hidden"], case["inter"]
    weights = _held(2 * i, h) + _held(h, i)
    if case["op"] == "feed_forward":
        return {"bytes": weights + 4 * n * h, "flops": 6 * n * h * i}
    rows = n * case["top_k"]
    return {"bytes": weights * min(case["experts"], rows) + 4 * n * h + 8 * rows, "flops": 6 * rows * h * i}


# --------------------------------------------------------------------------- the format
def _quantise(x):
    """[..., K] -> codes uint8 [..., K] of 0 .. 15 (8: the sign) and exponents uint8 [..., K / 32], 127 + e."""
    y = x.to(F32).unflatten(-1, (-1, BLOCK))
    top = y.abs().amax(-1)
    e = (torch.frexp(top)[1].to(torch.int32) - 3).clamp_(min=-127)                  # top = m 2^p, 0.5 <= m < 1
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    v = torch.ldexp(y, -e.unsqueeze(-1))
    a = v.abs()
    # a step of 1/2 below 2, of 1 below 4, of 2 above; 4, 6 and 7 codes lie below the sums
    code = torch.where(a < 2, (a * 2).round(), torch.where(a < 4, a.round() + 2, (a * 0.5).round() + 4)).clamp_(max=7)
    code = code.to(torch.uint8) + 8 * (v < 0).to(torch.uint8)
    return code.flatten(-2), (e + 127).to(torch.uint8)


def _values(codes, exponents):
    steps = torch.tensor(STEPS + tuple(-s for s in STEPS), dtype=F32, device=codes.device)
    y = steps[codes.int()].unflatten(-1, (-1, BLOCK))
    return torch.ldexp(y, (exponents.to(torch.int32) - 127).unsqueeze(-1)).flatten(-2)


# --------------------------------------------------------------------------- inputs
def _rows(g, n, k):
    """Activations: channels of uneven size, a few of them large."""
    size = torch.exp(0.6 * torch.randn(k, device=DEV, generator=g))
    return torch.randn(n, k, device=DEV, generator=g) * size


def _weight(g, m, k):
    return _quantise(torch.randn(m, k, device=DEV, generator=g) * k ** -0.5)


def _inputs(case, g):
    """What the case computes with: x, and for the others weights as codes and exponents, and what routing said."""
    n = case["tokens"]
    if case["op"] == "quantise":
        x = _rows(g, n, case["k"]).to(TYPES[case["dtype"]])
        return dict(x=x, **(_routing(case, g) if case["experts"] else {}))
    if case["op"] == "linear":
        x = _rows(g, n, case["k"]).to(BF16)
        bias = torch.randn(case["n_out"], device=DEV, generator=g).to(BF16) if case["bias"] else None
        return dict(x=x, w=_weight(g, case["n_out"], case["k"]), bias=bias)
    h, i = case["hidden"], case["inter"]
    x = _rows(g, n, h).to(BF16)
    if case["op"] == "feed_forward":
        return dict(x=x, gate=_weight(g, i, h), up=_weight(g, i, h), down=_weight(g, h, i))
    stacks = {}
    for name, m, k in (("gate", i, h), ("up", i, h), ("down", h, i)):
        parts = [_weight(g, m, k) for _ in range(case["experts"])]
        stacks[name] = tuple(torch.stack(p) for p in zip(*parts))
    return dict(x=x, **_routing(case, g), **stacks)


def _routing(case, g):
    """The experts of every token and their scores, some experts liked better than others."""
    n, experts = case["tokens"], case["experts"]
    logits = torch.randn(n, experts, device=DEV, generator=g) + 0.5 * torch.randn(experts, device=DEV, generator=g)
    chosen, ids = logits.topk(case["top_k"], dim=1)
    return dict(ids=ids.to(torch.int32).contiguous(), scores=torch.sigmoid(chosen).contiguous())


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(case=case, **_inputs(case, g))
    if "ids" in state and not own:                                  # rows of every expert, for the plain form's slices
        state["counts"] = torch.bincount(state["ids"].flatten().long(), minlength=case["experts"]).tolist()
    if own and case["op"] != "quantise":
        from hi_b200.kernels import ops

        # laid out once, when a model is loaded
        if case["op"] == "linear":
            state["w"] = ops.mx_pack_weight(*state["w"])
        else:
            gate, up = state.pop("gate"), state.pop("up")
            both = [ops.mx_interleave(a, b) for a, b in zip(gate, up)]
            state["gate_up"] = ops.mx_pack_weight(*both, glu=True)
            state["down"] = ops.mx_pack_weight(*state["down"])
    return state


# --------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    return {"quantise": _run_quantise, "linear": _run_linear, "feed_forward": _run_feed_forward,
            "experts": _run_experts}[case["op"]](case, state)


def _sorted_tokens(state):
    """The tokens' entries by expert, within one in their order."""
    return torch.argsort(state["ids"].flatten(), stable=True)


def _run_quantise(case, state):
    """The rows as the values they stand for."""
    x = state["x"]
    if own:
        from hi_b200.kernels import ops

        if case["experts"]:
            plan = ops.moe_plan(state["ids"], case["experts"])
            return ops.mx_values(ops.mx_quantize(x, plan, case["top_k"]), BF16)
        return ops.mx_values(ops.mx_quantize(x), BF16)
    if case["experts"]:
        x = x[_sorted_tokens(state) // case["top_k"]]
    return _values(*_quantise(x)).to(BF16)


def _run_linear(case, state):
    out = TYPES[case["out"]]
    if own:
        from hi_b200.parts.linear import linear

        return linear(state["x"], state["w"], out_dtype=out, bias=state["bias"])
    y = _values(*_quantise(state["x"])) @ _values(*state["w"]).t()
    if state["bias"] is not None:
        y = y + state["bias"].to(F32)
    return y.to(out)


def _unit(gate, up, limit):
    """silu(gate) * up, or with a limit the clamped unit."""
    if limit > 0:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit) + 1
        return gate / (1 + torch.exp(-1.702 * gate)) * up
    return gate / (1 + torch.exp(-gate)) * up


def _run_feed_forward(case, state):
    if own:
        from hi_b200.kernels import ops

        return ops.mx_linear(ops.mx_glu(state["x"], state["gate_up"], limit=case["limit"]), state["down"])
    x = _values(*_quantise(state["x"]))
    act = _unit(x @ _values(*state["gate"]).t(), x @ _values(*state["up"]).t(), case["limit"])
    return (_values(*_quantise(act)) @ _values(*state["down"]).t()).to(BF16)


def _run_experts(case, state):
    n, k = case["tokens"], case["top_k"]
    on_input = case["scale"] == "input"
    if own:
        from hi_b200.kernels import ops

        plan = ops.moe_plan(state["ids"], case["experts"])
        act = ops.mx_experts_glu(state["x"], plan, k, state["gate_up"], state["scores"] if on_input else None, limit=case["limit"])
        y = ops.mx_experts_linear(act, state["down"], plan)
        return ops.convert(ops.moe_combine(y, plan.slot_of_entry, None, n, k, None if on_input else state["scores"].view(-1)), BF16)
    order = _sorted_tokens(state)
    x = _values(*_quantise(state["x"]))[order // k]
    score = state["scores"].view(-1)[order].unsqueeze(1)
    parts, at = [], 0
    for e, count in enumerate(state["counts"]):
        rows = slice(at, at + count)
        at += count
        if not count:
            continue
        gate, up, down = (_values(state[name][0][e], state[name][1][e]) for name in ("gate", "up", "down"))
        s = score[rows] if on_input else 1.0
        act = _unit(s * (x[rows] @ gate.t()), s * (x[rows] @ up.t()), case["limit"])
        parts.append(_values(*_quantise(act)) @ down.t())
    y = torch.cat(parts)
    if not on_input:
        y = y * score
    out = torch.zeros((n, case["hidden"]), dtype=F32, device=DEV)
    back = torch.empty_like(y)
    back[order] = y                                                 # an entry's row in its place, a token's entries side by side
    return torch.sum(back.view(n, k, -1), dim=1, out=out).to(BF16)


# --------------------------------------------------------------------------- in 64 bits
def _exact_held(x):
    """The values that [..., K] stands for once it is quantised, in 64 bits: by the borders between neighbours."""
    y = x.to(F64).reshape(*x.shape[:-1], -1, BLOCK)
    top = y.abs().max(dim=-1, keepdim=True).values
    power = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    power = torch.where(torch.pow(2.0, power) > top, power - 1, power)              # (a logarithm next to a whole number)
    power = torch.where(torch.pow(2.0, power + 1) <= top, power + 1, power)
    unit = torch.pow(2.0, torch.clamp(power - 2, min=-127.0))
    a = (y / unit).abs()
    steps = torch.tensor(STEPS, dtype=F64, device=x.device)
    borders = (steps[1:] + steps[:-1]) / 2
    low = torch.searchsorted(borders, a.contiguous(), right=False)                  # a value on a border goes down ..
    high = torch.searchsorted(borders, a.contiguous(), right=True)                  # .. or up, to the even one of the two
    code = torch.where(low % 2 == 0, low, high)
    return torch.where(top > 0, torch.sign(y) * steps[code] * unit, torch.zeros_like(y)).reshape(x.shape)


def _exact_weight(codes, exponents):
    steps = torch.tensor(STEPS, dtype=F64, device=codes.device)
    sign = 1.0 - 2.0 * (codes >= 8).to(F64)
    unit = torch.pow(2.0, exponents.to(F64) - 127.0).repeat_interleave(BLOCK, dim=-1)
    return sign * steps[(codes % 8).long()] * unit


def _exact_unit(gate, up, limit):
    if limit > 0:
        gate = torch.minimum(gate, torch.full_like(gate, limit))
        return gate * torch.sigmoid(1.702 * gate) * (torch.clamp(up, min=-limit, max=limit) + 1.0)
    return gate * torch.sigmoid(gate) * up


def exact(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    given = _inputs(case, g)
    x = given["x"]
    if case["op"] == "quantise":
        if case["experts"]:
            entries = torch.sort(given["ids"].reshape(-1), stable=True).indices
            x = torch.index_select(x, 0, torch.div(entries, case["top_k"], rounding_mode="floor"))
        return _exact_held(x)
    held = _exact_held(x)
    if case["op"] == "linear":
        y = torch.mm(held, _exact_weight(*given["w"]).t())
        return y if given["bias"] is None else y + given["bias"].to(F64)
    if case["op"] == "feed_forward":
        gate, up = (torch.mm(held, _exact_weight(*given[name]).t()) for name in ("gate", "up"))
        return torch.mm(_exact_held(_exact_unit(gate, up, case["limit"])), _exact_weight(*given["down"]).t())
    out = torch.zeros((case["tokens"], case["hidden"]), dtype=F64, device=DEV)
    for e in range(case["experts"]):
        token, choice = torch.nonzero(given["ids"] == e, as_tuple=True)
        if not token.numel():
            continue
        score = given["scores"][token, choice].to(F64).unsqueeze(1)
        before, after = (score, 1.0) if case["scale"] == "input" else (1.0, score)
        gate, up = (before * torch.mm(held[token], _exact_weight(*(t[e] for t in given[name])).t()) for name in ("gate", "up"))
        act = _exact_held(_exact_unit(gate, up, case["limit"]))
        out.index_add_(0, token, after * torch.mm(act, _exact_weight(*(t[e] for t in given["down"])).t()))
    return out
