"""Engines whose weights are microscaled 4-bit floats: every product of their steps against float64 of what the codes stand for, captured
steps against eager ones, what is refused and what stays as it is."""
import pytest
import torch

import bezasun_configs
import fofisun_configs
import harness as h
import plain_mx
from tiny_configs import TINY_A, TINY_B

BF16 = torch.bfloat16


def test_options_that_are_refused():
    from hi_b200.config.registry import lookup
    from hi_b200.parts.model import Model

    def build(**kw):
        arch = lookup(TINY_A)
        return Model(arch.build_spec(arch.parse_config(TINY_A, None)), kw.pop("dtype", BF16), "cpu", **kw)

    assert build(weight_bits=4, weight_format="mxfp4").env.weight_format == "mxfp4"
    for kw in (dict(weight_bits=4, weight_format="fp4"), dict(weight_format=None), dict(weight_format="mxfp4"),
               dict(weight_bits=4, weight_format="mxfp4", dtype=torch.float32)):
        with pytest.raises(ValueError):
            build(**kw)


def _watch(monkeypatch, seen):
    """Checks of every product: rows are what the format says, sums are those of exact products."""
    from hi_b200.kernels import ops
    from test_mx import _check_unit, _near

    weights = {}

    def values(w):
        if id(w) not in weights:
            e, m, k = w.codes.shape[0], w.codes.shape[1], w.shape[-1]
            codes = torch.stack([w.codes & 15, w.codes >> 4], -1).view(e, m, k)
            s = w.scales.view(e, w.scales.shape[1], -1, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(e, w.scales.shape[1] * 128, -1)
            weights[id(w)] = (w, plain_mx.values(codes, s[:, :m, : k // 32].contiguous()))
        return weights[id(w)][1]

    def gate_up(v):
        v = v.view(v.shape[0], 2, 32, v.shape[1]) if v.dim() == 3 and v.shape[0] == 0 else v.unflatten(0, (-1, 2, 32))
        return v[:, 0].flatten(0, 1), v[:, 1].flatten(0, 1)

    def rows_of(x):
        if isinstance(x, ops.MxRows):
            return ops.mx_values(x, torch.float32).double()
        held = plain_mx.held(x)
        assert torch.equal(ops.mx_values(ops.mx_quantize(x), torch.float32).double(), held)
        return held

    linear, glu, experts_glu, experts_linear = ops.mx_linear, ops.mx_glu, ops.mx_experts_glu, ops.mx_experts_linear

    def checked_linear(x, weight, out_dtype=BF16, bias=None):
        y = linear(x, weight, out_dtype, bias)
        _near(y, rows_of(x), values(weight)[0], bias)
        seen["linear"] += 1
        return y

    def checked_glu(x, weight, limit=0.0):
        act = glu(x, weight, limit)
        _check_unit(rows_of(act), rows_of(x), *gate_up(values(weight)[0]), limit)
        seen["glu"] += 1
        return act

    def checked_experts_glu(x, plan, top_k, weight, scores=None, limit=0.0):
        act = experts_glu(x, plan, top_k, weight, scores, limit)
        entries, offsets = plan.sorted_entry.long(), plan.offsets.tolist()
        xs, got = rows_of(x)[entries // top_k], rows_of(act)
        for e in range(len(offsets) - 1):
            at = slice(offsets[e], offsets[e + 1])
            if at.start < at.stop:
                _check_unit(got[at], xs[at], *gate_up(values(weight)[e]), limit, None if scores is None else scores.view(-1)[entries[at]])
        seen["experts"] += 1
        return act

    def checked_experts_linear(rows, weight, plan):
        y = experts_linear(rows, weight, plan)
        offsets, xs = plan.offsets.tolist(), rows_of(rows)
        for e in range(len(offsets) - 1):
            at = slice(offsets[e], offsets[e + 1])
            if at.start < at.stop:
                _near(y[at], xs[at], values(weight)[e])
        return y

    for name, f in (("mx_linear", checked_linear), ("mx_glu", checked_glu), ("mx_experts_glu", checked_experts_glu),
                    ("mx_experts_linear", checked_experts_linear)):
        monkeypatch.setattr(ops, name, f)


CONFIGS = {"llama4": TINY_A, "two_experts": TINY_B["text_config"] | {"architectures": TINY_B["architectures"]}, "bezasun": bezasun_configs.BZ_B,
           "fofisun": fofisun_configs.FO_B}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CONFIGS))
def test_every_product_of_an_engine(name, monkeypatch):
    """Prompts, mixed steps and single tokens through models with dense feed-forwards, shared and routed experts."""
    from hi_b200.engine.core import Engine, StepEntry
    from hi_b200.kernels import ops

    cfg = CONFIGS[name]
    eng = Engine.from_config(cfg, seed=5, std=0.08, weight_bits=4, weight_format="mxfp4", kv_page_size=16, kv_cache_tokens=1024,
                             max_active_requests=3, use_cuda_graphs=False)
    seen = dict(linear=0, glu=0, experts=0)
    _watch(monkeypatch, seen)
    toks = [(37 * i * i + 11 * i + 5) % 128 for i in range(200)]
    out = [eng.step([StepEntry("a", toks[:140], [139])])]
    out += [eng.step([StepEntry("a", [toks[140]], [0]), StepEntry("b", toks[141:160], [18])])]
    out += [eng.step([StepEntry("a", [t], [0]), StepEntry("b", [t], [0])]) for t in toks[160:164]]
    assert all(torch.isfinite(o).all() for o in out) and seen["linear"] > 0 and seen["experts"] > 0, seen
    assert seen["glu"] > 0 or name in ("bezasun", "fofisun")          # their dense and shared units are others, or not multiples of 32
    ops.check_tc_status()


@pytest.mark.gpu
def test_captured_steps():
    """Steps that are replayed from a graph against eager ones."""
    from hi_b200.engine.core import Engine, StepEntry

    runs = []
    for graphs in (True, False):
        eng = Engine.from_config(dict(TINY_A), seed=5, std=0.08, weight_bits=4, weight_format="mxfp4", kv_page_size=16, kv_cache_tokens=1024,
                                 max_active_requests=3, use_cuda_graphs=graphs)
        toks = h.random_tokens(TINY_A, 60, seed=2)
        out = [eng.step([StepEntry("a", toks[:30], [29]), StepEntry("b", toks[30:50], [19])])]
        out += [eng.step([StepEntry("a", [t], [0]), StepEntry("b", [t], [0])]) for t in toks[50:]]
        runs.append(torch.cat([o.float() for o in out]))
        assert graphs == bool(eng._graphs)
    assert h.rel_err(runs[0].cpu(), runs[1].cpu()) <= 1e-3


@pytest.mark.gpu
def test_what_is_held_how():
    """Projections, feed-forwards, shared and routed experts in 4 bits; embeddings, the head, routers and norms as they were; generate and LLM
    take the option."""
    import hi_b200
    from hi_b200.engine.core import Engine
    from hi_b200.kernels import ops

    eng = Engine.from_config(dict(TINY_A), seed=1, weight_bits=4, weight_format="mxfp4", kv_page_size=16, kv_cache_tokens=256)
    moe = [l for l in eng.model.layers if hasattr(l.feed_forward, "w_router")]
    assert moe
    for layer in moe:
        assert isinstance(layer.mixer.w_qkv, ops.MxWeight) and isinstance(layer.feed_forward.w_gate_up, ops.MxWeight)
        assert layer.feed_forward.w_up is None and isinstance(layer.feed_forward.w_down, ops.MxWeight)
        assert isinstance(layer.feed_forward.shared.w_gate_up, ops.MxWeight) and layer.feed_forward.w_router.dtype == BF16
    eng = Engine.from_config(dict(TINY_A), seed=1, weight_bits=4, kv_page_size=16, kv_cache_tokens=256)
    assert isinstance(eng.model.layers[0].mixer.w_qkv, ops.FourBitWeight)
    llm = hi_b200.LLM(dict(TINY_A), random_seed=3, weight_bits=4, weight_format="mxfp4", kv_cache_bits=4, kv_cache_tokens=512, kv_page_size=16)
    outs = llm.generate([[1, 2, 3], [4, 5]], hi_b200.SamplingParams(max_tokens=4, ignore_eos=True))
    assert [len(o.token_ids) for o in outs] == [4, 4]
