"""The 4-bit cache where its neighbours could reach a request: tables of expanded pages, positions that the host and the device do not agree on,
reshaped scores against float64, portions beside requests and rows of other magnitudes."""
import math

import pytest
import torch

from plain_four_bit import quantise, values, visible

BF16 = torch.bfloat16
DEV = "cuda:0"


def _step(portions, nh, nkv, hd, page, **kw):
    from test_four_bit import Step

    return Step(portions, nh, nkv, hd, page, **kw)


def _reshaped(q, k, v, seen, positions, scale, cap=0.0, slopes=None, sink=None):
    """float64: scores cap tanh(scale q k / cap) - slope (position - key), softmax with the sink's term. Returns the result, the same with |v|, and
    scale times the largest sum |q| |k| of a row (what roundings of the keys are relative to)."""
    per = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(per, 1), v.double().repeat_interleave(per, 1)
    hidden = ~seen.any(0)
    k, v = k.masked_fill(hidden.view(-1, 1, 1), 0), v.masked_fill(hidden.view(-1, 1, 1), 0)
    s = torch.einsum("nhd,thd->nht", q, k) * scale
    size = (scale * torch.einsum("nhd,thd->nht", q.abs(), k.abs())).masked_fill(~seen.unsqueeze(1), 0).amax(-1, keepdim=True)
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        distance = positions.view(-1, 1).double() - torch.arange(k.shape[0], device=q.device).double()
        s = s - slopes.double().view(1, -1, 1) * distance.unsqueeze(1)
    s = s.masked_fill(~seen.unsqueeze(1), -math.inf)
    top = s.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink.double().view(1, -1, 1))
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink.double().view(1, -1, 1) - top)
    p = p / total
    return torch.einsum("nht,thd->nhd", p, v), torch.einsum("nht,thd->nhd", p, v.abs()), size


def _check_reshaped(step, s, got, mask, scale, cap, slopes=None, sink=None):
    """Keys rounded to bfloat16 (2^-8 of each, which moves a score by up to 2^-8 of scale sum |q| |k|, less under a cap) and a cap by fast functions
    (2^-20 of it): a weight against its sum is off by twice that; values and weights rounded to bfloat16, and the result."""
    a, b = step.cu[s], step.cu[s + 1]
    k, v = values(quantise(step.k[s])), values(quantise(step.v[s]))
    seen = visible(step.positions[a:b], k.shape[0], **mask)
    want, size, scores = _reshaped(step.q[a:b], k, v, seen, step.positions[a:b], scale, cap, slopes, sink)
    off = 2.0 ** -8 * scores + 2.0 ** -20 * cap
    tol = 2 * off * (1 + off) * size + 2.0 ** -8 * (2 * size + want.abs())
    diff = (got[a:b].double() - want).abs()
    assert (diff <= tol).all(), (s, float((diff / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 32), (64, 64)])
def test_a_table_of_expanded_pages_names_them_and_nothing_else(hd, page):
    from hi_b200.kernels import ops

    step = _step([(37, 0), (1, 200), (70, 3), (2, 63), (1, 500)], 4, 2, hd, page, seed=page).fill()
    ctx = step.ctx
    wide = torch.cat([step.table, torch.full_like(step.table[:1], 5)])            # a row behind the last request
    for chunk, window, keep, skip in ((0, 0, 0, False), (64, 0, 0, False), (0, 20, 0, True), (0, 20, 5, False), (100, 0, 0, True)):
        for given in (step.table, wide):
            k, _v, table = ops.expand_pages_4bit(step.pages, hd, given, ctx.cu_seqlens, step.positions, ctx.start_pos, ctx.n_new, chunk, window,
                                                 keep, skip)
            want, at = torch.full_like(given, -1), 0
            for s, (n, c) in enumerate(step.portions):
                if skip and n == 1:
                    continue
                low = c // chunk * chunk if chunk else max(0, c - window + 1) if window and not keep else 0
                count = (c + n - 1) // page - low // page + 1
                want[s, low // page: low // page + count] = torch.arange(at, at + count, dtype=torch.int32, device=DEV)
                at += count
            assert k.shape[0] == at and torch.equal(table, want)
    none = ops.expand_pages_4bit(step.pages, hd, step.table, ctx.cu_seqlens * 0, step.positions, ctx.start_pos, [0] * 5)[2]
    assert (none == -1).all()
    ops.check_tc_status()


@pytest.mark.gpu
@pytest.mark.parametrize("host", [[0, 0], [300, 380]])
def test_positions_that_the_device_does_not_have_are_found(host):
    """More pages on the device than the host asked for, and fewer: no entry names a page that is not there, and the step's check raises."""
    from hi_b200.kernels import ops

    step = _step([(1, 300), (1, 90)], 4, 2, 64, 64, seed=3).fill()
    k, _v, table = ops.expand_pages_4bit(step.pages, 64, step.table, step.ctx.cu_seqlens, step.positions, host, [1, 1])
    assert int(table.max()) < k.shape[0] and int(table.min()) == -1
    with pytest.raises(ops.KernelError, match="4-bit cache"):
        ops.check_tc_status()
    ops.expand_pages_4bit(step.pages, 64, step.table, step.ctx.cu_seqlens, step.positions, [300, 90], [1, 1])
    ops.check_tc_status()
    for kw in ({}, dict(chunk=64), dict(window=70)):              # positions before the first: no pages
        table = ops.expand_pages_4bit(step.pages, 64, step.table, step.ctx.cu_seqlens, torch.full_like(step.positions, -1000), [300, 90], [1, 1], **kw)[2]
        assert (table == -1).all()
        with pytest.raises(ops.KernelError, match="4-bit cache"):
            ops.check_tc_status()


@pytest.mark.gpu
@pytest.mark.parametrize("page,window", [(32, 100), (16, 90), (16, 37)])
def test_a_request_beside_one_that_is_not_finite(page, window):
    """Request 0 has groups of NaN on its first pages; request 1's window starts inside a tile of keys, behind pages that nobody needs."""
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages

    step = _step([(70, 10), (200, 260), (33, 400)], 8, 2, 64, page, seed=window)
    step.k[0][3], step.v[0][:20] = float("nan"), float("nan")
    step.fill()
    ctx, scale = step.ctx, 0.125
    slopes = torch.rand(8, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) * 0.02
    for cap, slope in ((20.0, None), (0.0, slopes), (5.0, slopes)):
        got = attend_over_four_bit_pages(step.q, step.pages, step.table, ctx, 8, 2, 64, 0, window, scale, softcap=cap, slopes=slope)
        ops.check_tc_status()
        for s in (1, 2):
            _check_reshaped(step, s, got, dict(window=window), scale, cap, slope)
    for one_tile in (False, True):
        got = ops.prefill_attention_4bit(step.q, step.pages, step.table, ctx.cu_seqlens, step.positions, ctx.start_pos, ctx.n_new, 0, window, scale,
                                         one_tile=one_tile)
        ops.check_tc_status()
        for s in (1, 2):
            _check_reshaped(step, s, got, dict(window=window), scale, 0.0)


RESHAPED = [
    ([(40, 100), (1, 70), (1, 900)], 64, {}),
    ([(130, 700), (20, 0), (1, 33)], 32, dict(window=90)),
    ([(1, 300), (1, 64), (1, 2000)], 64, dict(window=100)),
    ([(1, 300), (1, 64), (1, 129)], 16, dict(chunk=100)),
    ([(90, 333), (1, 10)], 16, dict(window=50, keep=20)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", RESHAPED, ids=lambda c: f"p{c[1]}n{len(c[0])}" + "".join(f"_{k}{v}" for k, v in c[2].items()))
def test_reshaped_scores_against_float64(case):
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages

    portions, page, mask = case
    step = _step(portions, 8, 2, 64, page, seed=page + len(portions)).fill()
    g = torch.Generator(device=DEV).manual_seed(2)
    slopes, sinks = torch.rand(8, device=DEV, generator=g) * 0.02, torch.randn(8, device=DEV, generator=g)
    for cap, slope, sink in ((20.0, None, None), (0.0, slopes, None), (3.0, slopes, sinks)):
        got = attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, 8, 2, 64, mask.get("chunk", 0), mask.get("window", 0), 0.125,
                                         softcap=cap, slopes=slope, sink_values=sink, keep=mask.get("keep", 0))
        ops.check_tc_status()
        for s in range(len(portions)):
            _check_reshaped(step, s, got, mask, 0.125, cap, slope, sink)


def _tiny(**kw):
    import bezasun_configs

    return bezasun_configs.config(131, 64, 1e-5, [bezasun_configs.attention(4, 2, 16, 16, 0.25, mlp=None, **kw)])


@pytest.mark.parametrize("bits", [4, 16])
def test_steps_whose_pages_are_expanded_are_not_captured(bits):
    """On the CPU: capped or biased scores over a 4-bit cache need the host's positions at every step; other steps do not."""
    from hi_b200.config.registry import lookup
    from hi_b200.parts.model import Model
    from tiny_configs import TINY_A

    def build(cfg):
        arch = lookup(cfg)
        return Model(arch.build_spec(arch.parse_config(cfg, None)), BF16, "cpu", cache_bits=bits)

    for cfg in (_tiny(softcap=20.0), _tiny()):
        model = build(cfg)
        mixers = [layer.mixer for layer in model.layers]
        assert all(m.softcap or m.distance_bias is not None for m in mixers)
        assert model.graph_safe == (bits == 16)
    assert build(TINY_A).graph_safe


@pytest.mark.gpu
def test_engine_steps_with_reshaped_scores(tmp_path):
    """Decoding over several pages and across their ends, two and more requests: graphs asked for and not, and a cache in bfloat16 beside them."""
    import bezasun_configs
    import harness as h
    from hi_b200.engine.core import Engine, StepEntry

    mdir = str(tmp_path / "m")
    bezasun_configs.write_model(mdir, _tiny(softcap=20.0), 4)
    toks, other = ([(7 * i + s) % 128 for i in range(160)] for s in (1, 5))
    runs = []
    for graphs, bits in ((True, 4), (False, 4), (False, 16)):
        eng = Engine.from_dir(mdir, kv_page_size=16, kv_cache_tokens=640, max_active_requests=4, kv_cache_bits=bits, use_cuda_graphs=graphs,
                              graph_context_bucket=128)
        out = [eng.step([StepEntry("a", toks[:70], [69])]), eng.step([StepEntry("b", other[:30], [29])])]
        for i in range(40):
            out.append(eng.step([StepEntry("a", [toks[70 + i]], [0]), StepEntry("b", [other[30 + i]], [0])]))
        assert not eng._graphs
        eng.snapshot()
        runs.append(torch.cat(out).float().cpu())
    assert torch.equal(runs[0], runs[1])
    # what four bits do to the keys and values of one small layer; a wrong page gives logits that have nothing to do with these
    assert runs[0].isfinite().all() and torch.corrcoef(torch.stack([runs[0].flatten(), runs[2].flatten()]))[0, 1] > 0.9


@pytest.mark.gpu
@pytest.mark.parametrize("hd,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("one_tile", [False, True])
def test_a_portion_does_not_depend_on_other_requests(hd, page, one_tile):
    """The same numbers, bit by bit, beside requests whose keys and values are 2^20 and 2^90 times as large or as small, beside rows that no
    request owns. With one of its own queries grown: those of its warp (32 rows, which follow their maxima together) to float16's rounding, the
    others bit by bit."""
    from hi_b200.kernels import ops
    from test_four_bit import _check_rows

    def run(grown, size, query=1.0):
        step = _step([(40, 100), (150, 0), (1, 70), (33, 64)], 8, 2, hd, page, seed=31)
        for s in grown:
            step.k[s], step.v[s] = step.k[s] * size, step.v[s] * size
        step.fill()
        q = step.q.clone()
        q[39] *= query
        q = torch.cat([q, torch.full_like(q[:5], 3e38)])          # rows behind the last request
        ctx = step.ctx
        out = ops.prefill_attention_4bit(q, step.pages, step.table, ctx.cu_seqlens, step.positions, ctx.start_pos, ctx.n_new, 0, 0, 0.09,
                                         one_tile=one_tile)
        ops.check_tc_status()
        if query != 1.0:
            step.q = q[:224]
            _check_rows(step, 0, out, {}, 0.09, None, False)
        return out

    want = run((), 1.0)
    for size in (2.0 ** 20, 2.0 ** -20, 2.0 ** 90, 2.0 ** -90):
        got = run((1, 2), size)
        assert torch.equal(got[:40], want[:40]) and torch.equal(got[191:224], want[191:224])
    for query in (2.0 ** 10, 2.0 ** 30):                          # (scores of 2^34: their maxima's own rounding is more than float16 holds)
        got = run((), 1.0, query)
        assert torch.equal(got[:32], want[:32]) and torch.equal(got[40:224], want[40:224])


@pytest.mark.gpu
@pytest.mark.parametrize("one_tile", [False, True])
@pytest.mark.parametrize("form", ["row", "values", "keys", "queries", "large", "small"])
def test_portions_of_uneven_sizes(form, one_tile):
    """Groups of a request's kv head whose sizes lie further apart than float16 holds: rows that some queries read and others do not, a kv head's first
    32 dims, queries large where the keys are small; all of them near the ends of bfloat16. As exact as over bfloat16 pages."""
    from hi_b200.kernels import ops

    step = _step([(100, 200), (70, 0)], 8, 2, 128, 64, seed=41)
    scale, window = 0.09, 64
    if form == "row":                       # outside the windows of the later tokens, on a page of theirs
        step.k[0][140] *= 2.0 ** 40
        step.v[0][141] *= 2.0 ** 40
    elif form == "values":
        step.v[0][:, :, :32] *= 2.0 ** -30
        step.v[1][::3] *= 2.0 ** -30
    elif form == "keys":
        step.k[0][:, :, :32] *= 2.0 ** -30
        step.k[1][:, :, 32:] *= 2.0 ** -30
    elif form == "queries":
        step.k[0][:, :, :32] *= 2.0 ** -30
        step.q[:100, :, :32] *= 2.0 ** 30
    elif form == "large":
        step.k, step.q = [k * 2.0 ** 110 for k in step.k], step.q * 2.0 ** -110
        step.v = [v * 2.0 ** 110 for v in step.v]
    else:
        step.k, step.q = [k * 2.0 ** -110 for k in step.k], step.q * 2.0 ** 110
        step.v = [v * 2.0 ** -110 for v in step.v]
    step.fill()
    ctx = step.ctx
    for mask in ({}, dict(window=window)):
        got = ops.prefill_attention_4bit(step.q, step.pages, step.table, ctx.cu_seqlens, step.positions, ctx.start_pos, ctx.n_new, 0,
                                         mask.get("window", 0), scale, one_tile=one_tile)
        ops.check_tc_status()
        for s in (0, 1):
            if form == "row" and s == 0:            # the tokens whose window lies behind the large rows: to the size of what they read
                late = _step([(95, 205), (70, 0)], 8, 2, 128, 64, seed=41)
                late.k, late.v, late.q, late.positions = step.k, step.v, step.q[5:], step.positions[5:]
                if mask:
                    _check_reshaped(late, 0, got[5:], mask, scale, 0.0)
            else:
                _check_reshaped(step, s, got, mask, scale, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,page", [(128, 64), (64, 32)])
@pytest.mark.parametrize("one_tile,shares", [(False, 1), (False, 3), (True, 1), (True, 3)])
def test_many_small_weights(hd, page, one_tile, shares):
    """One key of no value that weighs 2^26 times as much as each of 6,000 others: they are all that the result is made of. Keys, values and scores
    are held exactly; a weight in float16 is off by 2^-32 of the largest or 2^-11 of itself, the exponential by 2^-17, the result is rounded."""
    from hi_b200.kernels import ops

    step = _step([(150, 6000), (40, 300)], 4, 2, hd, page, seed=5)
    for s in (0, 1):
        step.k[s].zero_()
        step.k[s][0, :, 0] = 15.0
        step.v[s].fill_(1.0)
        step.v[s][0] = 0.0
    step.fill()
    step.q.zero_()
    step.q[:, :, 0] = 1.0
    scale = 26 * math.log(2) / 15
    ctx = step.ctx
    for sink in (None, torch.full((4,), 26 * math.log(2), device=DEV), torch.full((4,), 0.0, device=DEV)):
        got = ops.prefill_attention_4bit(step.q, step.pages, step.table, ctx.cu_seqlens, step.positions, ctx.start_pos, ctx.n_new, 0, 0, scale,
                                         key_splits=shares, sink_values=sink, one_tile=one_tile)
        ops.check_tc_status()
        for s in (0, 1):
            a, b = step.cu[s], step.cu[s + 1]
            others = step.positions[a:b].double() * 2.0 ** -26
            extra = 0.0 if sink is None else math.exp(float(sink[0]) - 26 * math.log(2))
            want = (others / (1 + others + extra)).view(-1, 1, 1)
            tol = want * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -16) + others.view(-1, 1, 1) * 2.0 ** -6
            assert ((got[a:b].double() - want).abs() <= tol).all(), (s, float(got[a:b].min()), float(want.min()))


def test_a_status_names_one_kernel():
    """On the CPU, from the sources: no two kernels report the same number, and those that have words of their own are what reports them."""
    import inspect
    import os
    import re

    from hi_b200.kernels import build, ops

    def numbers(name):
        with open(os.path.join(build.CSRC, name)) as f:
            text = f.read()
        found = set()
        for first, plus in re.findall(r"atomicExch\((?:\w+\.)?status, (\d+)( \+ i)?\)", text):
            found |= {int(first), int(first) + 1} if plus else {int(first)}
        for first, plus in re.findall(r"wait\([^;]*?, (\d+)( \+ i)?\);", text):           # waits that hand their number on
            found |= {int(first), int(first) + 1} if plus else {int(first)}
        return found

    product, pair, one = (numbers(f) for f in ("four_bit_gemm_tc.cu", "attention_prefill_pair.cu", "attention_prefill_tc.cu"))
    grouped, cache = numbers("grouped_gemm_tc.cu"), numbers("four_bit_cache.cu")
    assert {51, 57, 59, 60, 61, 71} <= pair and {11, 21, 24} <= one and cache == {33}
    kinds = [product, pair, one, grouped, cache, numbers("attention_decode_tma.cu"), numbers("recurrence_chunked.cu")]
    assert all(not a & b for i, a in enumerate(kinds) for b in kinds[:i])
    words = {int(n): w for n, w in re.findall(r'(\d+): "([^"]+)"', inspect.getsource(ops.check_tc_status))}
    assert {n for n, w in words.items() if w.startswith("4-bit product")} == product
    assert not (pair | one) & set(words)


def test_codes_of_more_than_four_bits_are_refused():
    from hi_b200.kernels import ops

    codes = torch.full((3, 64), 15, dtype=torch.uint8)
    scales = torch.ones(3, 2, dtype=BF16)
    ops.pack_weight(codes, scales)
    for wrong in (16, 255):
        codes[2, 63] = wrong
        with pytest.raises(ops.KernelError, match="0 .. 15"):
            ops.pack_weight(codes, scales)


NO_MASK = [dict(chunk=512, keep=5), dict(chunk=64, window=1000, keep=200)]


def test_pages_between_kept_tokens_and_a_window_are_not_asked_for():
    """On the CPU: the count grows with the window, not with the context; and with every page of the request where all are wanted."""
    from array import array

    from hi_b200.kernels import ops

    def total(start, n, page, chunk=0, window=0, keep=0, whole=0):
        starts, counts = array("i", start), array("i", n)
        return ops.lib().hb_expand_total(starts.buffer_info()[0], counts.buffer_info()[0], len(n), 1 << 24, page, chunk, window, keep, whole, 0)

    for start, n, page, window, keep in ((10_000_000, 20, 64, 1024, 4), (5000, 300, 16, 100, 70), (90, 40, 64, 64, 130), (200, 1, 32, 20, 33)):
        last, first = (start + n - 1) // page, (start - window + 1) // page
        kept = -(-keep // page)
        assert total([start], [n], page, window=window, keep=keep) == len(set(range(kept)) | set(range(first, last + 1)) - set(range(first)))
        assert total([start], [n], page, window=window, keep=keep, whole=1) == last + 1
    assert total([700, 40], [10, 0], 64) == total([700, 40], [10, 0], 64, keep=5) == 12
    for wrong in (dict(chunk=-1), dict(window=-1), dict(keep=-1), *NO_MASK):
        assert total([700], [10], 64, **wrong) == -1


@pytest.mark.parametrize("wrong", NO_MASK, ids=str)
def test_kept_tokens_beside_chunks_are_refused_by_the_entries(wrong):
    """On the CPU: the entry points look at the mask before anything is launched or read."""
    from hi_b200.kernels import ops

    some = torch.zeros(64, dtype=torch.int64)
    p = (some.data_ptr() + 15) // 16 * 16
    chunk, window, keep = wrong.get("chunk", 0), wrong.get("window", 0), wrong["keep"]
    lib = ops.lib()
    assert lib.hb_attention_decode_4bit(p, p, p, 4, p, p, p, 1, 8, 2, 64, 64, chunk, window, keep, 0.1, 0, None, 1, 1, 0, None, None, p, None, 1,
                                        None) == 1001
    assert lib.hb_expand_pages_4bit(p, p, 4, p, p, 1, 1, 64, chunk, window, keep, 1, 0, 2, 64, p, p, p, p, None) == 1001


@pytest.mark.gpu
@pytest.mark.parametrize("wrong", NO_MASK, ids=str)
def test_kept_tokens_beside_chunks_are_refused(wrong):
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages

    for portions in ([(1, 700), (1, 20)], [(40, 700), (20, 64)]):
        step = _step(portions, 8, 2, 64, 64).fill()
        for cap in (0.0, 8.0):
            with pytest.raises(ops.KernelError):
                attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, 8, 2, 64, wrong.get("chunk", 0), wrong.get("window", 0), 0.125,
                                           softcap=cap, keep=wrong["keep"])


KEPT = [
    ([(40, 3000), (150, 20), (1, 2000)], 64, dict(window=100, keep=4)),
    ([(40, 3000), (16, 64), (33, 700)], 16, dict(window=100, keep=70)),
    ([(40, 300), (150, 20)], 32, dict(window=90, keep=200)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", KEPT, ids=lambda c: f"p{c[1]}" + "".join(f"_{k}{v}" for k, v in c[2].items()))
def test_portions_with_kept_tokens(case):
    """Kept tokens in front of a window, more and fewer than a page, also where no page lies between them; what nobody may read is
    not finite."""
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages

    portions, page, mask = case
    step = _step(portions, 8, 2, 64, page, seed=page + len(portions))
    window, keep = mask["window"], mask["keep"]
    hidden = []
    for s, (n, c) in enumerate(portions):
        seen = visible(step.positions[step.cu[s]: step.cu[s + 1]], n + c, **mask)
        unseen = (~seen.any(0)).nonzero().flatten()
        whole = [int(p) for p in unseen if p // page * page + page <= n + c and (~seen.any(0))[p // page * page: p // page * page + page].all()]
        step.k[s][whole], step.v[s][whole] = float("nan"), float("nan")
        hidden.append(len(whole))
    assert any(hidden) or keep == 200
    step.fill()
    for s, (n, c) in enumerate(portions):                        # and their pages are given back
        seen = visible(step.positions[step.cu[s]: step.cu[s + 1]], n + c, **mask).any(0)
        for p in range((n + c) // page):
            if not seen[p * page: p * page + page].any():
                step.table[s, p] = -1
    for cap in (0.0, 8.0):
        got = attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, 8, 2, 64, 0, window, 0.125, softcap=cap, keep=keep)
        ops.check_tc_status()
        for s in range(len(portions)):
            if cap:
                _check_reshaped(step, s, got, mask, 0.125, cap)
            else:
                from test_four_bit import _check_rows

                rows = slice(step.cu[s], step.cu[s + 1])
                seen = visible(step.positions[rows], step.k[s].shape[0], **mask).any(0)
                k, v = step.k[s], step.v[s]
                step.k[s], step.v[s] = k.masked_fill(~seen.view(-1, 1, 1), 0), v.masked_fill(~seen.view(-1, 1, 1), 0)
                _check_rows(step, s, got, mask, 0.125, None, portions[s][0] == 1)
                step.k[s], step.v[s] = k, v


def test_pools_leave_room_for_the_pages_that_portions_expand():
    """On the CPU: every page of a layer's pool as bfloat16 keys and values, and the portions' queries, fit beside the pools, whatever fraction of the
    memory they may take; pools in 16 bits are as large as before."""
    from hi_b200.cache.device import bytes_per_token, plan_groups, pool_budget, pool_tokens_for_budget, pool_tokens_that_fit
    from hi_b200.config.registry import lookup
    from hi_b200.parts.model import Model
    from tiny_configs import TINY_A

    cfg = dict(TINY_A, head_dim=128, attention_chunk_size=1 << 20)
    arch = lookup(cfg)
    spec = arch.build_spec(arch.parse_config(cfg, None))
    for bits in (16, 4):
        model = Model(spec, BF16, "cpu", cache_bits=bits)
        _, group_of = plan_groups(model.cache_specs)
        cost = bytes_per_token(model.cache_specs, 2)
        for free in (1 << 26, 1 << 30, 5 << 30):
            for fraction in (0.5, 0.9, 1.0):
                args = (model.cache_specs, 2, free, fraction, model.scratch_bytes, model.scratch_per_token, 64, 2)
                tokens = pool_tokens_that_fit(*args)
                plain = pool_tokens_for_budget(model.cache_specs, 2, pool_budget(free, fraction, model.scratch_bytes), 64, 2)
                if bits == 16:
                    assert tokens == plain
                    continue
                need = max(each * tokens[group_of[slot]] for slot, each in model.scratch_per_token.items())
                assert all(model.scratch_per_token[slot] == 4 * cs.kv_heads * cs.head_dim for slot, cs in model.cache_specs.items() if cs.paged)
                taken = sum(c * t for c, t in zip(cost, tokens)) + need + model.scratch_bytes
                assert free - (1 << 20) <= taken <= free + (1 << 17) if tokens != plain else taken <= free + (1 << 17)
                assert pool_tokens_that_fit(*args, most_tokens=4096) == [min(t, 4096) for t in tokens]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,group", [(40, 256, 32), (300, 2112, 64), (33, 50048, 128), (17, 50048, 32)])
@pytest.mark.parametrize("tokens", [1, 8, 13, 16, 20])
def test_linear_of_inputs_that_are_large_or_infinite(m, k, group, tokens):
    """Infinite outputs where the definition has them, NaN where infinities of both signs meet or one meets a weight of zero; finite ones to the
    float32 sums' rounding (K steps of 2^-24 of all magnitudes; the weight's rounding to bfloat16 from 17 rows on). Other rows do not change."""
    from hi_b200.kernels import ops
    from plain_four_bit import weight_values

    g = torch.Generator(device=DEV).manual_seed(m + k + tokens)
    codes = torch.randint(0, 16, (m, k), device=DEV, generator=g).to(torch.uint8)
    scales = ((0.5 + torch.rand(m, k // group, device=DEV, generator=g)) * 0.2 * k ** -0.5).to(BF16)
    w = ops.pack_weight(codes, scales)
    x = torch.randn(tokens, k, device=DEV, generator=g).to(BF16)
    bias = torch.randn(m, device=DEV, generator=g).to(BF16)
    plain = ops.four_bit_linear(x, w, torch.float32, bias)
    changed = sorted({0, tokens // 2, tokens - 1})
    x[changed[0], k - 1] = math.inf
    if len(changed) > 1:
        x[changed[1], 5], x[changed[1], k // 2] = 2.0 ** 100, -(2.0 ** 90)
        x[changed[2], 3], x[changed[2], k - 30] = math.inf, -math.inf
    got = ops.four_bit_linear(x, w, torch.float32, bias)
    ops.check_tc_status()
    exact = weight_values(codes, scales)
    for t in range(tokens):
        if t not in changed:
            assert torch.equal(got[t], plain[t])
            continue
        products = x[t].double() * exact
        want = products.sum(1) + bias.double()
        finite = want.isfinite()
        assert torch.equal(got[t].isnan(), want.isnan()) and torch.equal(got[t][want.isinf()].double(), want[want.isinf()])
        tol = (k * 2.0 ** -24 + (2.0 ** -8 if tokens > 16 else 0.0)) * products.abs().sum(1) + 2.0 ** -23 * want.abs()
        assert ((got[t].double() - want).abs() <= tol)[finite].all()
    if tokens == 1:
        assert got.isinf().any()


@pytest.mark.gpu
def test_portions_of_more_tokens_than_queries_are_refused():
    from hi_b200.kernels import ops

    step = _step([(40, 100), (30, 0)], 8, 2, 64, 64, seed=7).fill()
    ctx = step.ctx
    call = lambda q, **kw: ops.prefill_attention_4bit(q, step.pages, step.table, ctx.cu_seqlens, step.positions, ctx.start_pos, ctx.n_new, 0, 0, 0.1, **kw)
    for q in (step.q[:69], step.q[0], step.q[:, :7].contiguous()):
        with pytest.raises(ops.KernelError):
            call(q)
    with pytest.raises(ops.KernelError):
        call(step.q, key_splits=0)
    call(step.q)
    ops.check_tc_status()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_with_queries_of_any_size(hd):
    """Keys times a power of two and queries divided by it give the same numbers bit by bit. Beside a head whose query is zero or not finite: so do
    other tokens and other kv heads; heads of the same one follow their maxima together, and stay within a decode step's roundings."""
    from hi_b200.kernels import ops
    from test_four_bit import _check_rows

    def run(e, change=None):
        step = _step([(1, 300), (1, 40), (1, 1000)], 16, 2, hd, 64, seed=51)
        step.k, q = [k * 2.0 ** e for k in step.k], step.q * 2.0 ** -e
        step.fill()
        if change is not None:
            q[1, 3], q[2, 9, 5] = 0.0, change
        out = ops.decode_attention_4bit(q, step.pages, step.table, step.seq, step.positions, 0, 0, hd ** -0.5, 1001)
        ops.check_tc_status()
        if change is not None:
            step.q = q
            _check_rows(step, 1, out, {}, hd ** -0.5, None, True)           # the token with a query of zeros
        return out

    want, largest = run(0), _step([(1, 300), (1, 40), (1, 1000)], 16, 2, hd, 64, seed=51).v[2]
    for e in (60, -60, 64, -64, 100, -100):
        assert torch.equal(run(e), want)
    for change in (math.inf, float("nan")):
        got = run(0, change)
        others = torch.ones(3, 16, dtype=torch.bool, device=DEV)
        others[1, :8] = others[2, 8:] = False
        assert torch.equal(got[others], want[others]) and got[2, 9].isnan().all()
        mates = [8, 10, 11, 12, 13, 14, 15]
        # either is within 2^-8 of the values' parts, up to 3 of the largest, and twice 2^-8 of itself
        assert ((got[2, mates].double() - want[2, mates].double()).abs() <= 2 * 2.0 ** -8 * 5 * values(quantise(largest)).abs().amax()).all()
