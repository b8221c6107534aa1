"""Serving in four bits, as cases to time and to compare: products with 4-bit weights and group scales, the append of keys and
values to a cache held in 4 bits, and attention over that cache.

A 4-bit weight is w[m, k] = scale[m, k // group] * (code[m, k] - 8), codes 0 .. 15, scales bfloat16. A cached row of a key/value
head is cut into groups of 32 dims, each x = scale * code + low, codes 0 .. 15, scale and low bfloat16, where low is the group's
least value and scale a fifteenth of its range.

A case is a dict of plain values; ``portions`` is a text "new@cached,new@cached,...": what every request of the step brings and
what the cache holds of it already. With ``own`` the framework's calls are made, else the plain forms below.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
PAGE = 64
GROUP = 32                       # dims of a cached row that share a scale
TEMPERATURE = (8192.0, 0.1)      # of the layers without rotation: q *= 1 + 0.1 ln(1 + floor((pos + 1) / 8192))
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    attention = dict(op="attention", heads=40, kv_heads=8, dim=128, chunk=0, window=0)
    return [
        # one request's token through a small projection: launches and latency
        dict(name="linear_1x2048x2048", op="linear", tokens=1, n_out=2048, k=2048, group=64, bias=False, out="bfloat16"),
        # eight requests' tokens through gate and up of a wide feed-forward: the weights are what moves
        dict(name="linear_8x16384x5120", op="linear", tokens=8, n_out=16384, k=5120, group=128, bias=False, out="bfloat16"),
        # one token through its down projection, the finest groups, unrounded sums
        dict(name="linear_1x5120x8192_f32", op="linear", tokens=1, n_out=5120, k=8192, group=32, bias=False, out="float32"),
        # a step of many requests and a short portion: an odd number of tokens, q, k and v at once, with a bias
        dict(name="linear_99x7168x5120", op="linear", tokens=99, n_out=7168, k=5120, group=64, bias=True, out="bfloat16"),
        # a prompt through gate and up
        dict(name="linear_2048x16384x5120", op="linear", tokens=2048, n_out=16384, k=5120, group=128, bias=False,
             out="bfloat16"),
        # a serving batch's next rows into the cache
        dict(name="append_64", op="append", heads=40, kv_heads=8, dim=128,
             portions=",".join(f"1@{200 + (i * 2477) % 3801}" for i in range(64))),
        # a prompt's rows, and a short one's beside it
        dict(name="append_prompts", op="append", heads=40, kv_heads=8, dim=128, portions="1987@0,61@0"),
        # a chat's next token: one request, a thousand keys
        dict(name="decode_1x1000", **attention, portions="1@999"),
        # a full serving batch's next tokens, contexts as uneven as requests are
        dict(name="decode_64_ragged", **attention, portions=",".join(f"1@{200 + (i * 2477) % 3801}" for i in range(64))),
        # one token over a long document, heads of 64, a sliding window's layer beside it would be short: this one sees it all
        dict(name="decode_1x131072", op="attention", heads=32, kv_heads=8, dim=64, chunk=0, window=0, portions="1@131071"),
        # a mixed step on a layer of 8,192-token chunks: later portions of long prompts beside decoding requests
        dict(name="mixed_chunked", op="attention", heads=40, kv_heads=8, dim=128, chunk=8192, window=0,
             portions="513@7000,1@8190,200@1234,1@500,1@3000,129@0,1@12000"),
        # a prompt's second portion under a sliding window
        dict(name="portion_window", op="attention", heads=32, kv_heads=8, dim=128, chunk=0, window=1024,
             portions="1500@2500"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["linear", "linear", "append", "decode", "decode", "mixed"])
    if op == "linear":
        group = rng.choice([32, 64, 128])
        k, n_out = group * max(1, round(_log(rng, 256, 8192) / group)), _log(rng, 64, 16384)
        tokens = _log(rng, 1, 2048)
        tokens = max(1, min(tokens, 2048 * 16384 * 5120 // (k * n_out)))
        return dict(op="linear", tokens=tokens, n_out=n_out, k=k, group=group, bias=rng.random() < 0.3,
                    out="float32" if tokens <= 16 and rng.random() < 0.4 else "bfloat16")
    heads, kv = rng.choice([(40, 8), (16, 4), (32, 8), (8, 2), (24, 24), (16, 1)])
    dim = rng.choice([64, 128, 128])
    if op == "append":
        parts, left = [], _log(rng, 1, 2048)
        while left > 0 and len(parts) < 48:
            n = min(left, rng.choice([1, 1, 1, _log(rng, 1, 2048)]))
            left -= n
            parts.append(f"{n}@{rng.choice([0, _log(rng, 1, 4000)])}")
        return dict(op="append", heads=heads, kv_heads=kv, dim=dim, portions=",".join(parts))
    mask = rng.choice(["", "", "chunk", "window"])
    case = dict(op="attention", heads=heads, kv_heads=kv, dim=dim, chunk=rng.choice([512, 8192]) if mask == "chunk" else 0,
                window=rng.choice([100, 1024, 4096]) if mask == "window" else 0)
    if op == "decode":
        n, longest = _log(rng, 1, 64), _log(rng, 1, 32768)
        if n * longest * kv * dim > 160000 * 1024:
            longest = max(1, 160000 * 1024 // (n * kv * dim))
        case["portions"] = ",".join(f"1@{rng.randint(longest // 3, longest)}" for _ in range(n))
        return case
    parts, left = [], 2048
    for _ in range(rng.choice([1, 1, 2, 3])):
        new = min(_log(rng, 2, 2048), left)
        if new < 2:
            break
        left -= new
        parts.append(f"{new}@{rng.choice([0, _log(rng, 1, 16384 if new < 1024 else 2048)])}")
    parts += [f"1@{_log(rng, 1, 8192)}" for _ in range(rng.choice([0, 0, 2, 5]))]
    case["portions"] = ",".join(parts)
    return case


def _portions(case):
    return [tuple(int(v) for v in p.split("@")) for p in case["portions"].split(",")]


def _first_visible(case, start):
    """The oldest position that a token at ``start`` or later may read."""
    if case["chunk"]:
        return start // case["chunk"] * case["chunk"]
    return max(0, start - case["window"] + 1) if case["window"] else 0


def work(case):
    if case["op"] == "linear":
        n, m, k = case["tokens"], case["n_out"], case["k"]
        weights = m * k // 2 + 2 * m * k // case["group"]
        out = n * m * (4 if case["out"] == "float32" else 2)
        return {"bytes": weights + 2 * n * k + out + (2 * m if case["bias"] else 0), "flops": 2 * n * m * k}
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    row = 2 * nkv * (hd // 2 + 4 * hd // GROUP)                         # a token's key and value rows in the cache
    portions = _portions(case)
    tokens = sum(n for n, _c in portions)
    if case["op"] == "append":
        pages = sum((c + n - 1) // PAGE - c // PAGE + 1 for n, c in portions)
        read_back = pages * PAGE * (row + 4 * nkv * hd)
        return {"bytes": tokens * ((nh + 2 * nkv) * hd * 2 + nh * hd * 2 + row) + read_back,
                "flops": 8 * tokens * 2 * nkv * hd + 2 * pages * PAGE * 2 * nkv * hd}
    keys = sum(c + n - _first_visible(case, c) for n, c in portions)
    pairs = 0
    for n, c in portions:
        if case["window"]:
            pairs += sum(min(p + 1, case["window"]) for p in range(c, c + n))
        elif case["chunk"]:
            pairs += sum(p % case["chunk"] + 1 for p in range(c, c + n))
        else:
            pairs += n * c + n * (n + 1) // 2
    return {"bytes": keys * row + 2 * tokens * nh * hd * 2, "flops": 4 * nh * hd * pairs}


# --------------------------------------------------------------------------- inputs
def _linear_inputs(case, g):
    n, m, k, group = case["tokens"], case["n_out"], case["k"], case["group"]
    x = torch.randn(n, k, device=DEV, generator=g).to(BF16)
    # codes of normal weights scaled by their group's largest value: mostly the middle, each group's extreme at an end
    codes = (torch.randn(m, k, device=DEV, generator=g) * 2.7).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    scales = ((0.5 + torch.rand(m, k // group, device=DEV, generator=g)) * 0.3 * k ** -0.5).to(BF16)
    bias = torch.randn(m, device=DEV, generator=g).to(BF16) if case["bias"] else None
    return x, codes, scales, bias


def _rows(case, g, count):
    """Keys with channels of uneven size and offset, as projections give them, and values; [count, kv_heads, dim] bfloat16."""
    nkv, hd = case["kv_heads"], case["dim"]
    rnd = lambda *shape: torch.randn(*shape, device=DEV, generator=g)
    k = rnd(count, nkv, hd) * torch.exp(0.5 * rnd(nkv, hd)) + 0.5 * rnd(nkv, hd)
    return k.to(BF16), rnd(count, nkv, hd).to(BF16)


def _quantise(x):
    """[..., dim] -> codes uint8 [..., dim], scale and low bfloat16 [..., dim / 32]."""
    y = x.to(F32).unflatten(-1, (-1, GROUP))
    low, high = y.amin(-1), y.amax(-1)
    scale = ((high - low) / 15.0).to(BF16)
    step = scale.to(F32).unsqueeze(-1)
    codes = torch.where(step > 0, ((y - low.unsqueeze(-1)) / step).round().clamp(0, 15), torch.zeros_like(y))
    return codes.to(torch.uint8).flatten(-2), scale, low.to(BF16)


def _values(codes, scale, low):
    y = codes.to(F32).unflatten(-1, (-1, GROUP))
    return (scale.to(F32).unsqueeze(-1) * y + low.to(F32).unsqueeze(-1)).flatten(-2)


def _tables(portions, g):
    """The step's tables as the engine lays them out: pages of a request anywhere in the pool."""
    n_new, start = [n for n, _c in portions], [c for _n, c in portions]
    cu = [0]
    for n in n_new:
        cu.append(cu[-1] + n)
    positions = torch.cat([torch.arange(c, c + n) for n, c in portions]).to(torch.int32).to(DEV)
    seq = torch.repeat_interleave(torch.arange(len(portions)), torch.tensor(n_new)).to(torch.int32).to(DEV)
    need = [-(-(n + c) // PAGE) for n, c in portions]
    order = torch.randperm(sum(need), device=DEV, generator=g).to(torch.int32)
    table = torch.zeros((len(portions), max(need)), dtype=torch.int32, device=DEV)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at: at + k]
        at += k
    return dict(cu=cu, positions=positions, seq=seq, table=table, pages=sum(need), n_new=n_new, start=start)


def _context(t):
    from hi_b200.parts.context import StepContext

    n_new, start, cu = t["n_new"], t["start"], t["cu"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    ctx = StepContext(n_tokens=cu[-1], n_seqs=len(n_new), tokens=torch.zeros(cu[-1], dtype=torch.int32, device=DEV),
                      positions=t["positions"], seq_of_token=t["seq"], cu_seqlens=i32(cu), slots=i32(list(range(len(n_new)))),
                      start_pos=start, n_new=n_new, slot_ids=list(range(len(n_new))), page_size=PAGE,
                      max_context=max(n + c for n, c in zip(n_new, start)))
    singles = [i for i, n in enumerate(n_new) if n == 1]
    if singles and len(singles) < len(n_new):
        ctx.decode_rows = torch.tensor([cu[i] for i in singles], dtype=torch.int64, device=DEV)
        ctx.decode_max_context = max(start[i] + 1 for i in singles)
    return ctx


def _pool(case, pages):
    """Pages of the 4-bit cache, nothing written yet."""
    from hi_b200.kernels import ops

    return torch.zeros((pages, case["kv_heads"], ops.four_bit_page_bytes(PAGE, case["dim"])), dtype=torch.uint8, device=DEV)


def _append(case, pool, qkv, t, positions, seq, heads, temperature):
    from hi_b200.kernels import ops

    return ops.qkv_post_4bit(qkv, heads, case["kv_heads"], case["dim"], positions, None, False, False, 1e-6, temperature, seq,
                             t["table"], pool)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "linear":
        x, codes, scales, bias = _linear_inputs(case, g)
        state = dict(case=case, x=x, bias=bias, codes=codes, scales=scales)
        if own:
            from hi_b200.kernels import ops

            state["weight"] = ops.pack_weight(codes, scales)     # laid out once, when a model is loaded
        return state
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    portions = _portions(case)
    t = _tables(portions, g)
    n = t["cu"][-1]
    q = torch.randn(n, nh, hd, device=DEV, generator=g).to(BF16)
    state = dict(case=case, t=t)
    if case["op"] == "append":
        k, v = _rows(case, g, n)
        state["qkv"] = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], dim=1).contiguous()
        if own:
            state["pool"], state["ctx"] = _pool(case, t["pages"]), _context(t)
        else:
            groups = (t["pages"], nkv, PAGE, hd // GROUP)
            for name in "kv":
                state[name] = (torch.zeros((t["pages"], nkv, PAGE, hd), dtype=torch.uint8, device=DEV),
                               torch.zeros(groups, dtype=BF16, device=DEV), torch.zeros(groups, dtype=BF16, device=DEV))
        return state
    state["q"] = q
    if own:
        state["pool"], state["ctx"] = _pool(case, t["pages"]), _context(t)
    else:
        state["cache"] = []
    for s, (new, cached) in enumerate(portions):
        k, v = _rows(case, g, new + cached)
        if not own:
            state["cache"].append((_quantise(k), _quantise(v)))
            continue
        for a in range(0, new + cached, 8192):
            b = min(a + 8192, new + cached)
            rows = torch.cat([k[a:b].flatten(1), k[a:b].flatten(1), v[a:b].flatten(1)], dim=1).contiguous()
            _append(case, state["pool"], rows, t, torch.arange(a, b, dtype=torch.int32, device=DEV),
                    torch.full((b - a,), s, dtype=torch.int32, device=DEV), nkv, None)
    return state


# --------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    return {"linear": _run_linear, "append": _run_append, "attention": _run_attention}[case["op"]](case, state)


def _run_linear(case, state):
    out = F32 if case["out"] == "float32" else BF16
    if own:
        from hi_b200.parts.linear import linear

        return linear(state["x"], state["weight"], out_dtype=out, bias=state["bias"])
    w = (state["codes"].to(F32) - 8.0).unflatten(1, (-1, case["group"])) * state["scales"].to(F32).unsqueeze(-1)
    y = state["x"].to(F32) @ w.flatten(1).t()
    if state["bias"] is not None:
        y = y + state["bias"].to(F32)
    return y.to(out)


def _touched(portions, table):
    """Pages that hold the step's new tokens, request by request."""
    return torch.cat([table[s, c // PAGE: (c + n - 1) // PAGE + 1] for s, (n, c) in enumerate(portions)]).long()


def _temperature(positions, dtype):
    floor_scale, attn_scale = TEMPERATURE
    return torch.log(torch.floor((positions.to(dtype) + 1.0) / floor_scale) + 1.0) * attn_scale + 1.0


def _run_append(case, state):
    """The step's rows go into the cache; q, and the pages that were written, as the values they stand for."""
    t, qkv = state["t"], state["qkv"]
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    if own:
        from hi_b200.kernels import ops

        ctx = state["ctx"]
        q = _append(case, state["pool"], qkv, t, t["positions"], t["seq"], nh, TEMPERATURE)
        # a window of one token: the pages from a request's first new token on
        k_pages, v_pages, _table = ops.expand_pages_4bit(state["pool"], hd, t["table"], ctx.cu_seqlens, t["positions"],
                                                         ctx.start_pos, ctx.n_new, window=1)
        return q, k_pages, v_pages
    n = qkv.shape[0]
    q, k, v = qkv.split([nh * hd, nkv * hd, nkv * hd], dim=1)
    q = (q.view(n, nh, hd).to(F32) * _temperature(t["positions"], F32).view(n, 1, 1)).to(BF16)
    page = t["table"][t["seq"].long(), (t["positions"] // PAGE).long()].long()
    row = (t["positions"] % PAGE).long()
    touched = _touched(_portions(case), t["table"])
    out = [q]
    for name, x in (("k", k), ("v", v)):
        for pool, part in zip(state[name], _quantise(x.reshape(n, nkv, hd))):
            pool[page, :, row] = part
        out.append(_values(*(pool[touched] for pool in state[name])).to(BF16))
    return tuple(out)


def _visible(case, positions, first, last):
    """[tokens, keys] which of the keys first .. last - 1 each token reads."""
    at = torch.arange(first, last, device=DEV)
    p = positions.long().unsqueeze(1)
    seen = at <= p
    if case["chunk"]:
        seen &= at >= p // case["chunk"] * case["chunk"]
    if case["window"]:
        seen &= at > p - case["window"]
    return seen


def _attend(case, q, k, v, positions, first):
    """q [n, heads, dim] over k, v [keys, kv_heads, dim] at positions first ..; in the type of its operands."""
    n, nh, hd = q.shape
    nkv = k.shape[1]
    seen = _visible(case, positions, first, first + k.shape[0])
    out = torch.empty_like(q)
    per = nh // nkv
    rows = max(1, (1 << 29) // (per * k.shape[0]))
    for h in range(nkv):
        for a in range(0, n, rows):
            heads = slice(h * per, (h + 1) * per)
            s = torch.einsum("nhd,td->hnt", q[a: a + rows, heads], k[:, h]) * hd ** -0.5
            s = s.masked_fill(~seen[a: a + rows], float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            out[a: a + rows, heads] = torch.einsum("hnt,td->nhd", p / p.sum(-1, keepdim=True), v[:, h])
    return out


def _run_attention(case, state):
    t = state["t"]
    if own:
        from hi_b200.parts.attention import attend_over_four_bit_pages

        return attend_over_four_bit_pages(state["q"], state["pool"], t["table"], state["ctx"], case["heads"], case["kv_heads"],
                                          case["dim"], case["chunk"], case["window"], case["dim"] ** -0.5)
    out = []
    for s, (_new, cached) in enumerate(_portions(case)):
        a, b = t["cu"][s], t["cu"][s + 1]
        first = _first_visible(case, cached)
        k, v = (_values(*(part[first:] for part in rows)) for rows in state["cache"][s])
        out.append(_attend(case, state["q"][a:b].to(F32), k, v, t["positions"][a:b], first))
    return torch.cat(out).to(BF16)


# --------------------------------------------------------------------------- in 64 bits
def _exact_cached(x):
    """The values that [..., dim] bfloat16 rows have once they are in the cache."""
    y = x.to(F64).reshape(*x.shape[:-1], -1, GROUP)
    low = y.min(dim=-1, keepdim=True).values
    step = ((y.max(dim=-1, keepdim=True).values - low) / 15).to(BF16).to(F64)
    codes = torch.clamp(torch.round((y - low) / torch.where(step > 0, step, torch.ones_like(step))), 0, 15)
    return torch.where(step > 0, low + step * codes, low).reshape(x.shape)


def exact(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "linear":
        x, codes, scales, bias = _linear_inputs(case, g)
        w = (codes.to(F64) - 8) * scales.to(F64).repeat_interleave(case["group"], dim=1)
        y = torch.mm(x.to(F64), w.t())
        return y if bias is None else y + bias.to(F64)
    nh, hd = case["heads"], case["dim"]
    portions = _portions(case)
    t = _tables(portions, g)
    n = t["cu"][-1]
    q = torch.randn(n, nh, hd, device=DEV, generator=g).to(BF16).to(F64)
    if case["op"] == "append":
        out = [q * _temperature(t["positions"], F64).view(n, 1, 1)]
        for x in _rows(case, g, n):
            pages, rows = [], _exact_cached(x)
            for s, (new, cached) in enumerate(portions):
                first, last = cached // PAGE, (cached + new - 1) // PAGE + 1
                line = torch.zeros(((last - first) * PAGE, *rows.shape[1:]), dtype=F64, device=DEV)
                line[cached - first * PAGE: cached + new - first * PAGE] = rows[t["cu"][s]: t["cu"][s + 1]]
                pages.append(line.view(last - first, PAGE, *rows.shape[1:]).transpose(1, 2))
            out.append(torch.cat(pages))
        return tuple(out)
    out = []
    for s, (new, cached) in enumerate(portions):
        k, v = (_exact_cached(x) for x in _rows(case, g, new + cached))
        per = nh // case["kv_heads"]
        for i in range(t["cu"][s], t["cu"][s + 1], 256):
            j = min(i + 256, t["cu"][s + 1])
            first = _first_visible(case, int(t["positions"][i]))
            last = int(t["positions"][j - 1]) + 1
            seen = _visible(case, t["positions"][i:j], first, last).unsqueeze(0)
            line = []
            for h in range(nh):
                scores = torch.mm(q[i:j, h], k[first:last, h // per].t()) / math.sqrt(hd)
                weights = torch.softmax(torch.where(seen[0], scores, torch.full_like(scores, -math.inf)), dim=-1)
                line.append(torch.mm(weights, v[first:last, h // per]))
            out.append(torch.stack(line, dim=1))
    return torch.cat(out)
