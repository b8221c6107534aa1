"""Calls at the edges of what the microscaled 4-bit operators take: tiles that end anywhere, by every form of the product."""
import pytest
import torch

import plain_mx
from test_mx import BF16, DEV, F32, _check_unit, _gen, _near, _rows, _weight


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
