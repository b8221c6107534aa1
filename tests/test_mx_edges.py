"""Calls at the edges of what the microscaled 4-bit operators take: tiles that end anywhere, by every form of the product."""
import pytest
import torch

import plain_mx
from test_mx import BF16, DEV, F32, _gen, _near, _rows, _weight


def _check_unit(act, x, gate, up, limit, score=None):
    """Values of a unit against 64 bits. Sums as in _near; the unit's slope in the gate is at most 1.2. Then, in units of 2^-23 of the result: the
    exponential 2 + 1.173 of its argument's magnitude and the division 2, as CUDA documents them, the clamped unit's 1.702 g, rounded twice, another
    1.702 |g| in the exponent, and half a unit each for 1 + e, u + 1 and the product: at most 6 + 3.7 |g|."""
    s = 1.0 if score is None else score.double().unsqueeze(1)
    g, u = s * (x @ gate.t()), s * (x @ up.t())
    tg, tu = (2.0 ** -16 * s * (x.abs() @ w.abs().t()) for w in (gate, up))
    want = plain_mx.unit(g, u, limit)
    wide = (u.abs() if limit == 0 else u.clamp(-limit, limit).abs() + 1) + tu
    tol = 1.2 * tg * wide + (g.abs() + tg) * tu + (6 + 3.7 * g.abs()) * 2.0 ** -23 * want.abs()
    assert plain_mx.is_quantised(act, want, tol)


def _plan_of(counts):
    """A plan of one expert a token, expert e for counts[e] of them, in no order."""
    from hi_b200.kernels import ops

    ids = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)).to(torch.int32)
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(sum(counts)))].to(DEV)
    return ops.moe_plan(ids.view(-1, 1).contiguous(), len(counts))


def _units(x, counts, plan, gate, up, limit=0.0, scores=None):
    """mx_experts_glu against 64 bits, expert by expert: the weight, the rows and their values."""
    from hi_b200.kernels import ops

    w = ops.mx_pack_weight(*(ops.mx_interleave(a, b) for a, b in zip(gate, up)), glu=True)
    act = ops.mx_experts_glu(x, plan, 1, w, scores, limit)
    values, entries, at = ops.mx_values(act, F32).double(), plan.sorted_entry.long(), 0
    for e, count in enumerate(counts):
        rows = slice(at, at + count)
        at += count
        if count:
            _check_unit(values[rows], plain_mx.held(x)[entries[rows]], plain_mx.values(gate[0][e], gate[1][e]), plain_mx.values(up[0][e], up[1][e]), limit,
                        None if scores is None else scores.view(-1)[entries[rows]])
    return w, act, values


@pytest.mark.gpu
@pytest.mark.parametrize("counts,i,k,form", [([250, 0, 131, 193], 4128, 288, 1256), ([100, 17, 1, 128, 33], 4128, 288, 1128), ([5, 30, 20], 6432, 64, 1064),
                                             ([700, 129, 1450], 8224, 2080, 0)])
def test_units_of_tiles_that_end_anywhere(counts, i, k, form):
    """Tiles whose last runs are not full, with further tiles behind them: lanes without a row go on with those that have one."""
    from hi_b200.kernels import ops

    assert ops.lib().hb_mx_gemm_form(sum(counts), len(counts), 2 * i, k, 1) == form
    g = _gen(i + k + len(counts))
    x, plan = _rows(g, sum(counts), k), _plan_of(counts)
    gate, up = _weight(g, len(counts), i, k), _weight(g, len(counts), i, k)
    w, act, values = _units(x, counts, plan, gate, up)
    down = _weight(g, len(counts), 41, i)
    y, at = ops.mx_experts_linear(act, ops.mx_pack_weight(*down), plan), 0
    for e, count in enumerate(counts):
        if count:
            _near(y[at: at + count], values[at: at + count], plain_mx.values(down[0][e], down[1][e]))
        at += count
    for _ in range(5):
        assert torch.equal(ops.mx_values(ops.mx_experts_glu(x, plan, 1, w), F32).double(), values)
    ops.check_tc_status()


@pytest.mark.gpu
@pytest.mark.parametrize("at", [0, 1, 2])
@pytest.mark.parametrize("h,i", [(8192, 96), (8192, 1024), (640, 8192), (5120, 8192)])
@pytest.mark.parametrize("limit", [0.0, 1.5])
def test_one_routed_row(at, h, i, limit):
    """One token through its expert, whose products' K a cluster of blocks shares: the unit's, the down product's, or both."""
    from hi_b200.kernels import ops

    forms = [ops.lib().hb_mx_gemm_form(1, 3, 2 * i, h, 1), ops.lib().hb_mx_gemm_form(1, 3, h, i, 0)]
    assert max(forms) >= 2000
    g, counts = _gen(h + i + at), [int(e == at) for e in range(3)]
    x, plan, gate, up, down = _rows(g, 1, h), _plan_of(counts), _weight(g, 3, i, h), _weight(g, 3, i, h), _weight(g, 3, h, i)
    scores = torch.rand(1, 1, device=DEV, generator=g) + 0.5
    for s in (None, scores):
        w, act, values = _units(x, counts, plan, gate, up, limit, s)
        y = ops.mx_experts_linear(act, ops.mx_pack_weight(*down), plan)
        _near(y, values, plain_mx.values(down[0][at], down[1][at]))
        out = ops.moe_combine(y, plan.slot_of_entry, None, 1, 1, scores.view(-1))
        assert ((out.double() - y.double() * scores.double()).abs() <= 2 * 2.0 ** -24 * y.double().abs() * scores.double()).all()
    ops.check_tc_status()


@pytest.mark.gpu
@pytest.mark.parametrize("counts,i,h,form", [([3, 0, 20, 9], 96, 288, 1064), ([100, 17, 1, 128, 33], 160, 288, 1128), ([250, 3, 131, 193], 4128, 288, 1256),
                                             ([700, 129, 1450], 8224, 2080, 0)])
def test_clamped_experts(counts, i, h, form):
    """The clamped unit by expert in every form, gates and ups on both sides of the limit, with the score on what an expert reads and without."""
    from hi_b200.kernels import ops

    assert ops.lib().hb_mx_gemm_form(sum(counts), len(counts), 2 * i, h, 1) == form
    g = _gen(i + h + len(counts))
    x, plan, gate, up = _rows(g, sum(counts), h), _plan_of(counts), _weight(g, len(counts), i, h), _weight(g, len(counts), i, h)
    for scores in (None, torch.rand(sum(counts), 1, device=DEV, generator=g) + 0.5):
        _units(x, counts, plan, gate, up, 1.0, scores)
    ops.check_tc_status()


# ---------------------------------------------------------------- entries without an expert
@pytest.mark.gpu
@pytest.mark.parametrize("n,experts,top_k", [(1, 4, 2), (9, 3, 1), (40, 16, 4), (200, 5, 2), (700, 64, 3), (33, 2, 1)])
@pytest.mark.parametrize("some", [True, False])
def test_entries_without_an_expert(n, experts, top_k, some):
    """Ids that name no expert (a padded batch's): the plan's slots, rows and results of the others; or no entry has one."""
    from hi_b200.kernels import ops

    g, h, i = _gen(n + experts), 416, 160
    ids = torch.randn(n, experts, device=DEV, generator=g).topk(top_k, 1).indices.to(torch.int32)
    none = torch.rand(n, top_k, device=DEV, generator=g) < (0.4 if some else 2.0)
    none[-1] = True
    ids[none] = torch.tensor([-1, experts, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32, device=DEV)[torch.arange(int(none.sum()), device=DEV) % 4]
    plan = ops.moe_plan(ids.contiguous(), experts)
    flat = ids.view(-1).long()
    real = (flat >= 0) & (flat < experts)
    count = int(real.sum())
    order = torch.argsort(torch.where(real, flat, torch.full_like(flat, experts)), stable=True)[:count]
    assert int(plan.offsets[-1]) == count and torch.equal(plan.sorted_entry[:count].long(), order)
    assert (plan.sorted_entry[count:] == 0).all() and (plan.slot_of_entry[~real] == -1).all()
    assert torch.equal(plan.slot_of_entry[order].long(), torch.arange(count, device=DEV))
    x, scores = _rows(g, n, h), torch.rand(n, top_k, device=DEV, generator=g)
    held = plain_mx.held(x)
    assert torch.equal(ops.mx_values(ops.mx_quantize(x, plan, top_k), F32)[:count].double(), held[order // top_k])
    gate, up, down = _weight(g, experts, i, h), _weight(g, experts, i, h), _weight(g, experts, h, i)
    act = ops.mx_experts_glu(x, plan, top_k, ops.mx_pack_weight(*(ops.mx_interleave(a, b) for a, b in zip(gate, up)), glu=True), scores)
    y = ops.mx_experts_linear(act, ops.mx_pack_weight(*down), plan)
    values, offsets = ops.mx_values(act, F32).double(), plan.offsets.tolist()
    for e in range(experts):
        rows = slice(offsets[e], offsets[e + 1])
        if rows.start < rows.stop:
            entries = order[rows]
            _check_unit(values[rows], held[entries // top_k], plain_mx.values(gate[0][e], gate[1][e]), plain_mx.values(up[0][e], up[1][e]), 0.0,
                        scores.view(-1)[entries])
            _near(y[rows], values[rows], plain_mx.values(down[0][e], down[1][e]))
    terms = torch.zeros(n * top_k, h, dtype=torch.float64, device=DEV)
    terms[order] = y[:count].double() * scores.view(-1)[order].double().unsqueeze(1)
    terms = terms.view(n, top_k, h)
    out = ops.moe_combine(y, plan.slot_of_entry, None, n, top_k, scores.view(-1))
    odd = ops.moe_combine(y[:, : h - 1].contiguous(), plan.slot_of_entry, None, n, top_k, scores.view(-1))
    # a term's rounding and each of k sums, 2^-24 of all magnitudes each
    for got in (out, odd):
        want = terms[..., : got.shape[1]]
        assert ((got.double() - want.sum(1)).abs() <= (top_k + 1) * 2.0 ** -24 * want.abs().sum(1)).all() and not got[-1].any()
    ops.check_tc_status()


# ---------------------------------------------------------------- what is not a number
@pytest.mark.gpu
@pytest.mark.parametrize("n,i,k,form", [(3, 64, 288, 1064), (33, 64, 288, 1064), (100, 96, 512, 1128), (384, 4096, 1056, 1192), (195, 6016, 288, 1256),
                                        (500, 4128, 1056, 0), (1, 1024, 9248, 2000), (17, 1024, 9248, 2000)])
@pytest.mark.parametrize("limit", [0.0, 1.5])
def test_units_of_what_is_not_a_number(n, i, k, form, limit):
    """A row with an infinity or with what is not a number leaves as one that is none, whichever the unit, and so does a block of features whose
    weights have one; all others are what they are without."""
    from hi_b200.kernels import ops

    taken = ops.lib().hb_mx_gemm_form(n, 1, 2 * i, k, 1)
    assert taken >= 2000 if form == 2000 else taken == form           # 2000: some blocks share K, how many goes by the device
    g = _gen(n + i + k)
    x, gate, up = _rows(g, n, k), _weight(g, i, k), _weight(g, i, k)
    pack = lambda a, b: ops.mx_pack_weight(*(ops.mx_interleave(c, d) for c, d in zip(a, b)), glu=True)
    before = ops.mx_values(ops.mx_glu(x, pack(gate, up), limit), F32)
    assert before.isfinite().all()
    bad = torch.zeros(n, i, dtype=torch.bool, device=DEV)
    x[n // 2, 5], x[n - 1, k - 1] = float("inf"), float("nan")
    bad[n // 2], bad[n - 1] = True, True
    for rows in (x, ops.mx_quantize(x)):
        got = ops.mx_values(ops.mx_glu(rows, pack(gate, up), limit), F32)
        assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], before[~bad])
    gate[1][3, 0], up[1][i - 1, k // 32 - 1] = 255, 255
    bad[:, :32], bad[:, i - 32:] = True, True
    got = ops.mx_values(ops.mx_glu(x, pack(gate, up), limit), F32)
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], before[~bad])
    ops.check_tc_status()


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [0.0, 1.5])
@pytest.mark.parametrize("scale", [None, "input"])
def test_experts_of_what_is_not_a_number(limit, scale):
    """The same for tokens among their experts, and for a score that is not a number."""
    from hi_b200.kernels import ops

    g, counts, h, i = _gen(11), [40, 0, 7, 200], 288, 96
    n, plan = sum(counts), _plan_of(counts)
    x, gate, up, down = _rows(g, n, h), _weight(g, 4, i, h), _weight(g, 4, i, h), _weight(g, 4, 64, i)
    scores = torch.rand(n, 1, device=DEV, generator=g) if scale else None
    w, wd = ops.mx_pack_weight(*(ops.mx_interleave(a, b) for a, b in zip(gate, up)), glu=True), ops.mx_pack_weight(*down)

    def run():
        act = ops.mx_experts_glu(x, plan, 1, w, scores, limit)
        return ops.moe_combine(ops.mx_experts_linear(act, wd, plan), plan.slot_of_entry, None, n, 1)

    before = run()
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    x[3, 7], x[100, 287] = -float("inf"), float("nan")
    bad[3], bad[100] = True, True
    if scale:
        scores[50] = float("nan")
        bad[50] = True
    got = run()
    assert before.isfinite().all() and got[bad].isnan().all() and torch.equal(got[~bad], before[~bad])
    ops.check_tc_status()


# ---------------------------------------------------------------- refusals
def _packed(*shape, glu=False):
    """A weight on the host."""
    from hi_b200.kernels import ops

    return ops.mx_pack_weight(*plain_mx.quantise(torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape)))), glu=glu)


def _host_plan(n, experts):
    from hi_b200.kernels import ops

    z = lambda m: torch.zeros(m, dtype=torch.int32)
    return ops.MoePlan(z(experts + 1), z(n), z(n), z(experts + 1))


def test_scores_that_want_gradients_are_refused():
    from hi_b200.kernels import ops

    x, w, scores = torch.zeros(4, 64, dtype=BF16), _packed(3, 128, 64, glu=True), torch.rand(4, 2, requires_grad=True)
    with pytest.raises(ops.KernelError, match="no gradients"):
        ops.mx_experts_glu(x, _host_plan(8, 3), 2, w, scores)
    with torch.no_grad(), pytest.raises(ops.KernelError, match="CUDA"):            # what is refused then is the host's tensor
        ops.mx_experts_glu(x, _host_plan(8, 3), 2, w, scores)


def test_what_is_not_rows_is_refused():
    """Rows that are not quantised, or are already, where the others are asked for; plans of no expert a token; sizes that an int does not hold."""
    from hi_b200.kernels import ops

    x, w, wg = torch.zeros(4, 64, dtype=BF16), _packed(3, 128, 64), _packed(3, 128, 64, glu=True)
    rows, plan = ops.MxRows(x, 4, 64), _host_plan(4, 3)
    for call in (lambda: ops.mx_values(x), lambda: ops.mx_experts_linear(x, w, plan), lambda: ops.mx_quantize(rows), lambda: ops.mx_quantize(rows, plan, 1),
                 lambda: ops.mx_experts_glu(rows, plan, 1, wg), lambda: ops.MxRows(torch.empty(0, device="meta"), 2 ** 31, 32),
                 lambda: ops.MxRows(torch.empty(0, device="meta"), 1, 2 ** 31),
                 lambda: ops.MxWeight(torch.empty(2, 2 ** 30, 16, dtype=torch.uint8, device="meta"),
                                      torch.empty(2, 2 ** 23, 2, 512, dtype=torch.uint8, device="meta"), (2, 2 ** 30, 32))):
        with pytest.raises(ops.KernelError):
            call()


@pytest.mark.gpu
def test_plans_of_no_expert_a_token_are_refused():
    from hi_b200.kernels import ops

    x, plan, w = torch.zeros(1, 64, dtype=BF16, device=DEV), _plan_of([1, 0, 0]), ops.mx_pack_weight(*_weight(_gen(1), 3, 128, 64), glu=True)
    for top_k in (0, -1):
        with pytest.raises(ops.KernelError):
            ops.mx_quantize(x, plan, top_k)
        with pytest.raises(ops.KernelError):
            ops.mx_experts_glu(x, plan, top_k, w)
