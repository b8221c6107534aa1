"""Rows in microscaled 4-bit floats and their products with such weights, against plain forms in float64."""
import pytest
import torch

import plain_mx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(g, n, k, dtype=BF16):
    return (torch.randn(n, k, device=DEV, generator=g) * torch.exp(0.7 * torch.randn(k, device=DEV, generator=g))).to(dtype)


def _weight(g, *shape):
    return plain_mx.quantise(torch.randn(*shape, device=DEV, generator=g) * shape[-1] ** -0.5)


def _plan(g, n, experts, top_k):
    from hi_b200.kernels import ops

    ids = torch.randn(n, experts, device=DEV, generator=g).topk(top_k, 1).indices.to(torch.int32).contiguous()
    return ids, ops.moe_plan(ids, experts)


# ---------------------------------------------------------------- quantisation
@pytest.mark.parametrize("n,k", [(1, 32), (3, 256), (128, 288), (129, 5120), (300, 96), (2, 13312)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantise(n, k, dtype):
    """Codes and exponents are the format's, bit by bit (a value on a border, a block of zeros, the smallest numbers and the largest among
    them); blocks past K are zero."""
    from hi_b200.kernels import ops

    x = _rows(_gen(n + k), n, k + 16, dtype)[:, :k]
    x[0, :8] = torch.tensor([0.25, -0.75, 1.25, 1.75, 2.5, -3.5, 5.0, 7.0], device=DEV, dtype=dtype)
    x[0, 8:32] = 0.1
    x[-1, -32:] = 0 if n % 2 else 2.0 ** -132
    if n > 2:
        x[1, :32] = 3e38 if dtype == F32 else torch.finfo(BF16).max
        x[2, :16] *= 2.0 ** -100
        x[2, 16:32] *= 2.0 ** -110
    got = ops.mx_quantize(x)
    codes, exps = plain_mx.quantise(x)
    want = plain_mx.values(codes, exps)
    assert torch.equal(ops.mx_values(got, F32).double(), want) and torch.equal(ops.mx_values(got).double(), want)
    packed = ops.mx_pack_weight(codes, exps)
    c = lambda t: torch.where(t & 7 != 0, t & 15, t & 7) + torch.where(t & 112 != 0, t & 240, t & 112)      # the sign of a zero says nothing
    assert torch.equal(c(got.codes), c(packed.codes[0]))
    tile = lambda t: t.view(-1, t.shape[-2], 32, 4, 4).permute(0, 3, 2, 1, 4).flatten(3).flatten(0, 2)      # rows in order, their scales
    assert torch.equal(tile(got.scales)[:n], tile(packed.scales[0])[:n])


def test_quantise_what_is_not_finite():
    """Infinities and what is not a number: their block is not a number, the others are what they were."""
    from hi_b200.kernels import ops

    x = _rows(_gen(3), 40, 320)
    x[0, 5], x[1, 64], x[39, 319], x[7, 300] = float("inf"), -float("inf"), float("nan"), float("nan")
    got, want = ops.mx_values(ops.mx_quantize(x), F32).double(), plain_mx.held(x)
    assert want.isnan().sum() == 4 * 32 and torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))


@pytest.mark.parametrize("n,experts,top_k", [(1, 4, 2), (5, 128, 1), (130, 3, 3), (500, 16, 2), (64, 64, 6), (9, 1, 1)])
def test_quantise_sorted(n, experts, top_k):
    """Rows in their experts' order, some experts without any, some with more than a tile."""
    from hi_b200.kernels import ops

    g = _gen(n + experts)
    x = _rows(g, n, 416)
    _ids, plan = _plan(g, n, experts, top_k)
    got = ops.mx_values(ops.mx_quantize(x, plan, top_k), F32).double()
    assert torch.equal(got, plain_mx.held(x[plan.sorted_entry[: n * top_k].long() // top_k]))


def test_quantise_weight():
    from hi_b200.kernels import ops

    for shape in ((100, 96), (128, 512), (3, 130, 288), (1, 64, 64), (16, 128, 256)):
        w = torch.randn(shape, device=DEV, generator=_gen(sum(shape))).to(BF16)
        got, want = ops.mx_quantize_weight(w), ops.mx_pack_weight(*plain_mx.quantise(w))
        m = shape[-2]
        rows = lambda t: t.view(t.shape[0], t.shape[1], -1, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).flatten(1, 3)[:, :m]
        assert got.shape == want.shape and torch.equal(got.codes & 119, want.codes & 119) and torch.equal(rows(got.scales), rows(want.scales))


# ---------------------------------------------------------------- products
def _near(got, x, w, bias=None):
    """Products of two codes and two powers of two are exact. Float32 sums: a step of 64 k may drop 2^-23 of the largest of its 65 terms from
    each; the running sum of n steps of such terms is about sqrt(64 n) of them, all magnitudes together 64 n times 0.6: over 160 steps 9 sqrt(n) 2^-23,
    under 2^-16 of all magnitudes. Then the result's own rounding."""
    want, size = x @ w.transpose(-1, -2), x.abs() @ w.abs().transpose(-1, -2)
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    tol = 2.0 ** -16 * size + (2.0 ** -8 if got.dtype == BF16 else 2.0 ** -23) * want.abs()
    assert got.shape == want.shape and ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("m,k", [(1, 32), (64, 64), (127, 256), (128, 288), (129, 2048), (300, 8192), (2000, 544), (5120, 1024)])
@pytest.mark.parametrize("n", [1, 8, 17, 64, 100, 128, 129, 300])
def test_linear(m, k, n):
    """Tiles of rows and features that are not full, k that ends inside a stage and inside a chunk of scales, one row to several tiles."""
    from hi_b200.kernels import ops
    from hi_b200.parts.linear import linear

    g = _gen(m + k + n)
    x = _rows(g, n, k + 8)[:, :k]
    codes, exps = _weight(g, m, k)
    bias = torch.randn(m, device=DEV, generator=g).to(BF16)
    w = ops.mx_pack_weight(codes, exps)
    xv, wv = plain_mx.held(x), plain_mx.values(codes, exps)
    y = linear(x, w, out_dtype=F32)
    _near(y, xv, wv)
    _near(linear(x, w, out_dtype=F32, bias=bias), xv, wv, bias)
    assert torch.equal(linear(x, w), y.to(BF16)) and torch.equal(ops.mx_linear(ops.mx_quantize(x), w), y.to(BF16))
    _near(linear(x, w, bias=bias), xv, wv, bias)
    ops.check_tc_status()


@pytest.mark.parametrize("m,k,n", [(128, 8192, 5), (600, 10272, 9), (5120, 8192, 1), (1000, 8192, 33), (2048, 9248, 17), (300, 13312, 70)])
def test_linear_of_blocks_that_share_k(m, k, n):
    """Shares of unlike length, the last one short; every block finishes some rows, or has none to finish."""
    from hi_b200.kernels import ops

    assert ops.lib().hb_mx_gemm_form(n, 1, m, k, 0) >= 2000
    g = _gen(m + k + n)
    x, (codes, exps) = _rows(g, n, k), _weight(g, m, k)
    bias = torch.randn(m, device=DEV, generator=g).to(BF16)
    w, xv, wv = ops.mx_pack_weight(codes, exps), plain_mx.held(x), plain_mx.values(codes, exps)
    y = ops.mx_linear(x, w, F32, bias)
    _near(y, xv, wv, bias)
    assert torch.equal(ops.mx_linear(x, w, bias=bias), y.to(BF16)) and torch.equal(ops.mx_linear(ops.mx_quantize(x), w, F32, bias), y)
    if m % 64 == 0:
        act = ops.mx_values(ops.mx_glu(x, ops.mx_pack_weight(codes, exps, glu=True), 1.5), F32).double()
        gate, up = (wv.view(-1, 2, 32, k)[:, i].flatten(0, 1) for i in (0, 1))
        _check_unit(act, xv, gate, up, 1.5)
    ops.check_tc_status()


@pytest.mark.parametrize("m,k,n,rows", [(8200, 1056, 257, 192), (8192, 1056, 384, 192), (5120, 2080, 513, 192), (12032, 544, 190, 192), (12000, 544, 150, 192),
                                         (12032, 544, 193, 256), (8256, 1056, 500, 256), (8200, 1056, 460, 256)])
def test_linear_of_large_tiles(m, k, n, rows):
    """Tiles of up to 192 and 256 rows: second tiles that begin in the middle of a tile of scales, last ones of a few rows, sums that share columns."""
    from hi_b200.kernels import ops

    g = _gen(m + k + n)
    x, (codes, exps) = _rows(g, n, k), _weight(g, m, k)
    bias = torch.randn(m, device=DEV, generator=g).to(BF16)
    w, xv, wv = ops.mx_pack_weight(codes, exps), plain_mx.held(x), plain_mx.values(codes, exps)
    assert ops.lib().hb_mx_gemm_form(n, 1, m, k, 0) == 1000 + rows
    y = ops.mx_linear(x, w, F32, bias)
    _near(y, xv, wv, bias)
    assert torch.equal(ops.mx_linear(x, w, bias=bias), y.to(BF16))
    if m % 64 == 0:
        act = ops.mx_glu(x, ops.mx_pack_weight(codes, exps, glu=True), 1.5)
        gate, up = (wv.view(-1, 2, 32, k)[:, i].flatten(0, 1) for i in (0, 1))
        values = ops.mx_values(act, F32).double()
        _check_unit(values, xv, gate, up, 1.5)
        down = _weight(g, 40, m // 2)
        _near(ops.mx_linear(act, ops.mx_pack_weight(*down), F32), values, plain_mx.values(*down))
    ops.check_tc_status()


@pytest.mark.parametrize("m,k,n", [(16400, 5152, 2221), (16385, 4800, 2147), (24576, 5120, 1500)])
def test_linear_of_many_rows(m, k, n):
    """Pairs of blocks: several tiles a pair, tiles that are not full in rows, features and k, an odd number of features."""
    from hi_b200.kernels import ops

    assert ops.lib().hb_mx_gemm_form(n, 1, m, k, 0) == 0
    g = _gen(m + k + n)
    x, (codes, exps) = _rows(g, n, k), _weight(g, m, k)
    bias = torch.randn(m, device=DEV, generator=g).to(BF16)
    w, xv, wv = ops.mx_pack_weight(codes, exps), plain_mx.held(x), plain_mx.values(codes, exps)
    y = ops.mx_linear(x, w, F32, bias)
    _near(y, xv, wv, bias)
    assert torch.equal(ops.mx_linear(x, w, bias=bias), y.to(BF16)) and torch.equal(ops.mx_linear(ops.mx_quantize(x), w, F32, bias), y)
    ops.check_tc_status()


@pytest.mark.parametrize("limit", [0.0, 1.5])
def test_glu_of_many_rows(limit):
    from hi_b200.kernels import ops

    i, k, n = 8224, 5152, 2221
    assert ops.lib().hb_mx_gemm_form(n, 1, 2 * i, k, 1) == 0
    g = _gen(i)
    x, gate, up = _rows(g, n, k), _weight(g, i, k), _weight(g, i, k)
    w = ops.mx_pack_weight(*(ops.mx_interleave(a, b) for a, b in zip(gate, up)), glu=True)
    act = ops.mx_glu(x, w, limit)
    values = ops.mx_values(act, F32).double()
    _check_unit(values, plain_mx.held(x), plain_mx.values(*gate), plain_mx.values(*up), limit)
    down = _weight(g, 100, i)
    _near(ops.mx_linear(act, ops.mx_pack_weight(*down), F32), values, plain_mx.values(*down))       # blocks past its end are zeros
    ops.check_tc_status()


def test_linear_scales():
    """Powers of two over their whole range, and blocks that are not numbers: rows and columns that read them, no others."""
    from hi_b200.kernels import ops

    g = _gen(9)
    x = _rows(g, 150, 320, F32) * torch.pow(2.0, torch.randint(-60, 60, (150, 1), device=DEV, generator=g))
    codes, exps = _weight(g, 200, 320)
    exps = (exps.int() + torch.randint(-60, 60, (200, 1), device=DEV, generator=g)).to(torch.uint8)
    x[17, 3], exps[100, 9], exps[199, 0] = float("nan"), 255, 255
    y = ops.mx_linear(x, ops.mx_pack_weight(codes, exps), F32).double()
    bad = torch.zeros(150, 200, dtype=torch.bool, device=DEV)
    bad[17], bad[:, 100], bad[:, 199] = True, True, True
    assert torch.equal(y.isnan(), bad)
    xv, wv = plain_mx.held(x).nan_to_num(0), plain_mx.values(codes, exps).nan_to_num(0)
    off = (y - xv @ wv.t()).abs() - 2.0 ** -16 * (xv.abs() @ wv.abs().t())
    assert (off.masked_fill(bad, 0) <= 0).all()
    ops.check_tc_status()


# ---------------------------------------------------------------- the gated unit
def _check_unit(act, x, gate, up, limit, score=None):
    from hi_b200.kernels import ops

    s = 1.0 if score is None else score.double().unsqueeze(1)
    g, u = s * (x @ gate.t()), s * (x @ up.t())
    tg, tu = (2.0 ** -16 * s * (x.abs() @ w.abs().t()) for w in (gate, up))
    want = plain_mx.unit(g, u, limit)
    wide = (u.abs() if limit == 0 else u.clamp(-limit, limit).abs() + 1) + tu        # the unit's slopes: at most 1.2 in the gate
    tol = 1.2 * tg * wide + (g.abs() + tg) * tu + 2.0 ** -19 * want.abs()
    assert plain_mx.is_quantised(act, want, tol)


@pytest.mark.parametrize("i,k", [(32, 32), (64, 288), (96, 512), (160, 1024), (1024, 2080)])
@pytest.mark.parametrize("n", [1, 16, 100, 128, 260])
@pytest.mark.parametrize("limit", [0.0, 1.5])
def test_glu_and_down(i, k, n, limit):
    """The unit's result is quantised from its float32 value; the down product takes it as it is, blocks past its end among them."""
    from hi_b200.kernels import ops

    g = _gen(i + k + n)
    x = _rows(g, n, k)
    gate, up, down = _weight(g, i, k), _weight(g, i, k), _weight(g, 96, i)
    w = ops.mx_pack_weight(*(ops.mx_interleave(a, b) for a, b in zip(gate, up)), glu=True)
    act = ops.mx_glu(x, w, limit=limit)
    assert act.shape == (n, i)
    values = ops.mx_values(act, F32).double()
    _check_unit(values, plain_mx.held(x), plain_mx.values(*gate), plain_mx.values(*up), limit)
    _near(ops.mx_linear(act, ops.mx_pack_weight(*down), F32), values, plain_mx.values(*down))
    ops.check_tc_status()


@pytest.mark.parametrize("n,experts,top_k,h,i", [(1, 4, 1, 64, 32), (8, 16, 1, 512, 96), (64, 64, 6, 256, 160), (300, 3, 2, 288, 256),
                                                (700, 5, 1, 1056, 64), (40, 128, 4, 96, 64), (500, 384, 2, 64, 32), (130, 1, 1, 128, 128), (70, 2, 2, 2080, 64), (900, 3, 1, 544, 96), (12000, 4, 1, 5152, 4128)])
@pytest.mark.parametrize("scale", ["input", "output"])
def test_experts(n, experts, top_k, h, i, scale):
    """A token through its experts and back: experts without rows, with less than a tile and with several, the score before or after."""
    from hi_b200.kernels import ops

    g = _gen(n + experts + h)
    x = _rows(g, n, h)
    ids, plan = _plan(g, n, experts, top_k)
    scores = torch.rand(n, top_k, device=DEV, generator=g)
    gate, up, down = _weight(g, experts, i, h), _weight(g, experts, i, h), _weight(g, experts, h, i)
    w = ops.mx_pack_weight(*(ops.mx_interleave(a, b) for a, b in zip(gate, up)), glu=True)
    wd = ops.mx_pack_weight(*down)
    act = ops.mx_experts_glu(x, plan, top_k, w, scores if scale == "input" else None)
    y = ops.mx_experts_linear(act, wd, plan)
    values = ops.mx_values(act, F32).double()
    entries = plan.sorted_entry.long()
    xv = plain_mx.held(x)[entries // top_k]
    offsets = plan.offsets.tolist()
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        _check_unit(values[a:b], xv[a:b], plain_mx.values(gate[0][e], gate[1][e]), plain_mx.values(up[0][e], up[1][e]), 0.0,
                    scores.view(-1)[entries[a:b]] if scale == "input" else None)
        _near(y[a:b], values[a:b], plain_mx.values(down[0][e], down[1][e]))
    out = ops.moe_combine(y, plan.slot_of_entry, None, n, top_k, None if scale == "input" else scores.view(-1))
    want = torch.zeros(n * top_k, h, dtype=torch.float64, device=DEV)
    want[entries] = y.double() * (1.0 if scale == "input" else scores.view(-1)[entries].double().unsqueeze(1))
    want = want.view(n, top_k, h)
    # a term is its product's rounding off, 2^-24 of it, and each of k sums 2^-24 of a partial sum, which all magnitudes bound: (k + 1) 2^-24 of those
    assert ((out.double() - want.sum(1)).abs() <= (top_k + 1) * 2.0 ** -24 * want.abs().sum(1)).all()
    ops.check_tc_status()


def test_edges():
    """No rows; a weight alone on its stream; results that do not depend on the rows beside; a second call."""
    from hi_b200.kernels import ops

    g = _gen(2)
    w = ops.mx_pack_weight(*_weight(g, 256, 512))
    wg = ops.mx_pack_weight(*_weight(g, 256, 512), glu=True)
    assert ops.mx_linear(torch.empty(0, 512, dtype=BF16, device=DEV), w).shape == (0, 256)
    assert ops.mx_glu(torch.empty(0, 512, dtype=BF16, device=DEV), wg).shape == (0, 128)
    assert ops.mx_values(ops.mx_quantize(torch.empty(0, 512, dtype=BF16, device=DEV))).shape == (0, 512)
    x = _rows(g, 200, 512)
    y = ops.mx_linear(x, w, F32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = ops.mx_linear(x, w, F32)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z) and torch.equal(y[:150], ops.mx_linear(x[:150].float(), w, F32))
    wide = torch.zeros(200, 1026, dtype=BF16, device=DEV)
    wide[:, 513: 1025] = x                                             # rows that start at an odd place
    assert torch.equal(y, ops.mx_linear(wide[:, 513: 1025], w, F32)) and torch.equal(y, ops.mx_linear(x.t().contiguous().t(), w, F32))
    ops.check_tc_status()


def test_captured():
    """Calls in a graph, replayed with other inputs; two graphs in turn and side by side on two streams; the same results as eager ones."""
    from hi_b200.kernels import ops

    g = _gen(6)
    w = ops.mx_pack_weight(*_weight(g, 640, 1024))
    gate, up, down = _weight(g, 8, 128, 1024), _weight(g, 8, 128, 1024), _weight(g, 8, 1024, 128)
    wg, wd = ops.mx_pack_weight(*(ops.mx_interleave(a, b) for a, b in zip(gate, up)), glu=True), ops.mx_pack_weight(*down)

    def step(x, ids, scores):
        plan = ops.moe_plan(ids, 8)
        y = ops.mx_experts_linear(ops.mx_experts_glu(x, plan, 2, wg, scores), wd, plan)
        return ops.mx_linear(x, w), ops.moe_combine(y, plan.slot_of_entry, None, x.shape[0], 2)

    def inputs(n, seed):
        h = _gen(seed)
        return _rows(h, n, 1024), torch.randn(n, 8, device=DEV, generator=h).topk(2, 1).indices.int().contiguous(), torch.rand(n, 2, device=DEV, generator=h)

    graphs = []
    for n in (3, 150):
        static = inputs(n, 1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((n, static, graph, out, torch.cuda.Stream()))
    for seed in (2, 3, 4):
        for n, static, graph, out, stream in graphs:
            for a, b in zip(static, inputs(n, seed)):
                a.copy_(b)
        torch.cuda.synchronize()
        for n, static, graph, out, stream in graphs:
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for n, static, graph, out, stream in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, step(*inputs(n, seed))))
    ops.check_tc_status()


def test_a_row_depends_on_itself():
    """A token's results are the same whichever tokens stand beside it: the same bits where the form is, else to the float32 sums (2^-16 of all
    magnitudes each; a weight is 0.08 at most)."""
    from hi_b200.kernels import ops

    g = _gen(8)
    x, w = _rows(g, 2100, 5120), ops.mx_pack_weight(*_weight(g, 16384, 5120))
    whole = ops.mx_linear(x, w, F32)
    size = plain_mx.held(x[:3]).abs() @ plain_mx.values(*plain_mx.quantise(torch.full((1, 5120), 0.08, device=DEV))).abs().t()
    for n in (1, 40, 100, 300):
        assert ((ops.mx_linear(x[:n], w, F32)[:1].double() - whole[:1].double()).abs() <= 2.0 ** -15 * size[:1]).all()
    assert torch.equal(ops.mx_linear(x[1: 2100], w, F32)[:900], whole[1: 901])


def test_refusals():
    from hi_b200.kernels import ops

    g = _gen(4)
    w, wg = ops.mx_pack_weight(*_weight(g, 128, 256)), ops.mx_pack_weight(*_weight(g, 128, 256), glu=True)
    we, weg = ops.mx_pack_weight(*_weight(g, 3, 128, 256)), ops.mx_pack_weight(*_weight(g, 3, 128, 256), glu=True)
    x = _rows(g, 10, 256)
    ids, plan = _plan(g, 10, 3, 2)
    other = _plan(g, 10, 3, 2)[1]
    rows = ops.mx_quantize(x, plan, 2)
    scores = torch.rand(10, 2, device=DEV)
    many = ops.mx_pack_weight(*_weight(g, 385, 64, 256), glu=True)
    ids_many, plan_many = _plan(g, 10, 385, 2)
    for call in (lambda: ops.mx_experts_glu(x, plan_many, 2, many), lambda: ops.mx_linear(x, wg), lambda: ops.mx_glu(x, w), lambda: ops.mx_linear(x, we), lambda: ops.mx_linear(rows, w),
                 lambda: ops.mx_linear(x[:, :224], w), lambda: ops.mx_linear(x.half(), w), lambda: ops.mx_quantize(x[:, :40]),
                 lambda: ops.mx_linear(x, w, torch.float16), lambda: ops.mx_linear(x, w, bias=torch.zeros(127, dtype=BF16, device=DEV)),
                 lambda: ops.mx_linear(x, w, bias=torch.zeros(128, device=DEV)), lambda: ops.mx_linear(x[0], w),
                 lambda: ops.mx_experts_glu(x, plan, 2, we), lambda: ops.mx_experts_glu(x, plan, 1, weg), lambda: ops.mx_experts_glu(x, plan, 2, wg),
                 lambda: ops.mx_experts_glu(x, plan, 2, weg, scores[:9]), lambda: ops.mx_experts_glu(x, plan, 2, weg, scores.to(BF16)),
                 lambda: ops.mx_experts_linear(rows, we, other), lambda: ops.mx_experts_linear(ops.mx_quantize(x), we, plan),
                 lambda: ops.mx_experts_linear(rows, w, plan), lambda: ops.mx_quantize(x.float().requires_grad_()),
                 lambda: ops.mx_values(rows, torch.float16), lambda: ops.mx_quantize(x, plan, 3)):
        with pytest.raises(ops.KernelError):
            call()


@pytest.mark.parametrize("m,k", [(1, 32), (100, 288), (640, 1024), (7168, 5120), (300, 10240), (20000, 544), (128, 10272), (2048, 8192)])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16])
def test_rows_quantised_on_the_way(m, k, n):
    """Up to 16 rows, which the product's blocks quantise themselves: the same bits as rows that are quantised first; several tiles a block, shares of K,
    rows that lie apart, values on borders and such that are not finite."""
    from hi_b200.kernels import ops

    g = _gen(m + k + n + 3)
    for dtype in (BF16, F32):
        x = _rows(g, n, k + 24, dtype)[:, 8: 8 + k]
        x[0, :8] = torch.tensor([0.25, -0.75, 1.25, 1.75, 2.5, -3.5, 5.0, 7.0], device=DEV, dtype=dtype)
        if n > 2:
            x[1, 5], x[2, :32] = float("inf"), 0
        w = ops.mx_pack_weight(*_weight(g, m, k))
        bias = torch.randn(m, device=DEV, generator=g).to(BF16)
        bits = lambda t: t.view(torch.int16 if t.dtype == BF16 else torch.int32)
        for kind in (BF16, F32):
            assert torch.equal(bits(ops.mx_linear(x, w, kind, bias)), bits(ops.mx_linear(ops.mx_quantize(x), w, kind, bias)))
        if m % 64 == 0:
            w = ops.mx_pack_weight(*_weight(g, m, k), glu=True)
            a, b = (ops.mx_values(ops.mx_glu(v, w, 1.5), F32) for v in (x, ops.mx_quantize(x)))
            assert torch.equal(a.nan_to_num(99), b.nan_to_num(99))
    ops.check_tc_status()
