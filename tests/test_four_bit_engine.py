"""Engines that hold weights and cache in four bits: every attention call of their steps against float64 over the rows that lie in
the pages, their keys against the bfloat16 cache's, captured steps against eager ones, weights against the values they stand for,
and what is refused."""
import pytest
import torch

import bezasun_configs
import fidatar_configs
import harness as h
from plain_four_bit import GROUP, attention, quantise, unpack_weight, values, visible, weight_values
from tiny_configs import TINY_A

BF16 = torch.bfloat16


def test_options_that_are_refused():
    """On the CPU: a model says at once what its layers do not have in four bits."""
    from hi_b200.config.registry import lookup
    from hi_b200.parts.model import Model
    from vinurax_configs import VX_A

    def build(cfg, dtype=BF16, **kw):
        arch = lookup(cfg)
        return Model(arch.build_spec(arch.parse_config(cfg, None)), dtype, "cpu", **kw)

    model = build(TINY_A, cache_bits=4, weight_bits=4)
    assert all(cs.bits == 4 and cs.head_dim == 64 for cs in model.cache_specs.values())
    assert all(cs.bits == 16 and cs.head_dim == 16 for cs in build(TINY_A, weight_bits=4).cache_specs.values())
    with pytest.raises(ValueError, match="cache is not built in 4 bits"):
        build(VX_A, cache_bits=4)
    for kw in (dict(cache_bits=8), dict(weight_bits=3), dict(weight_group=16), dict(dtype=torch.float32, cache_bits=4),
               dict(dtype=torch.float32, weight_bits=4)):
        with pytest.raises(ValueError):
            build(TINY_A, **kw)
    wide = dict(TINY_A, head_dim=192)
    with pytest.raises(ValueError, match="heads of up to 128"):
        build(wide, cache_bits=4)


@pytest.mark.parametrize("option", [("--weight-bits", "4"), ("--kv-cache-bits", "4")])
def test_the_float32_reference_takes_no_four_bits(option, tmp_path):
    from hi_b200.cli import main

    with pytest.raises(SystemExit, match="four bits"):
        main(["run", str(tmp_path / "model"), "--tokens", "1,2,3", "--cpu", *option])


def test_a_cached_token_takes_five_eighths_of_a_byte_a_number():
    from hi_b200.cache.device import bytes_per_token
    from hi_b200.parts.spec import CacheSpec

    assert bytes_per_token({0: CacheSpec(8, 128, bits=4), 1: CacheSpec(8, 128, bits=4)}, 2) == [2 * 8 * 160]
    assert bytes_per_token({0: CacheSpec(8, 128), 1: CacheSpec(4, 64, window=("chunk", 64), bits=4)}, 2) == [8 * 128 * 4, 4 * 80]


@pytest.mark.gpu
def test_weights_stand_for_their_values(tmp_path):
    """An engine that quantises as it loads beside one that loads the values the codes stand for. In products of up to 16 tokens the one
    takes the exact values, the other their rounding to bfloat16; else they are the same."""
    from hi_b200.engine.core import Engine, StepEntry
    from hi_b200.kernels import ops

    cfg = dict(TINY_A, use_qk_norm=False)
    mdir = h.make_model(str(tmp_path / "m"), cfg, seed=3)
    weights = h.read_weights(mdir)
    changed = {}
    for name, w in weights.items():
        if any(k in name for k in ("q_proj", "k_proj", "v_proj", "o_proj", "shared_expert")):
            changed[name] = weight_values(*unpack_weight(ops.quantize_weight(w, 32)), torch.float32).to(BF16)
    assert len(changed) == 2 * 7
    other = h.make_model(str(tmp_path / "v"), cfg, seed=3, overrides=changed)
    toks = h.random_tokens(cfg, 150, seed=1)
    runs = []
    for d, kw in ((mdir, dict(weight_bits=4, weight_group=32)), (other, {})):
        eng = Engine.from_dir(d, kv_page_size=16, kv_cache_tokens=512, max_active_requests=2, **kw)
        out = [eng.step([StepEntry("a", toks[:100], list(range(100)))])]
        out += [eng.step([StepEntry("a", [t], [0])]) for t in toks[100:110]]
        out += [eng.step([StepEntry("a", toks[110:130], list(range(20))), StepEntry("b", toks[130:], [19])])]
        runs.append(torch.cat(out).float().cpu())
        if kw:
            layer = eng.model.layers[0]
            assert isinstance(layer.mixer.w_qkv, ops.FourBitWeight) and isinstance(layer.feed_forward.shared.w_down, ops.FourBitWeight)
    assert h.rel_err(runs[0], runs[1]) <= h.TOL_BF16


def _watch(monkeypatch, seen):
    """Checks of every append and every attention call of an engine's steps."""
    from hi_b200.kernels import ops
    from hi_b200.parts import attention as parts

    post, attend = ops.qkv_post_4bit, parts.attend_over_four_bit_pages

    def checked_post(qkv, nh, nkv, hd, positions, inv_freq, interleaved, qk_norm, eps, temperature, seq, table, kv_pages, write=True,
                     qw=None, kw=None, first=False, dim=0, mul=1.0, keys_as_values=False):
        q = post(qkv, nh, nkv, hd, positions, inv_freq, interleaved, qk_norm, eps, temperature, seq, table, kv_pages, write, qw, kw, first,
                 dim, mul, keys_as_values)
        page = kv_pages.shape[2] * 4 // (5 * hd)
        k16, v16 = (torch.zeros(kv_pages.shape[0], nkv, page, hd, dtype=BF16, device=qkv.device) for _ in range(2))
        want = ops.qkv_post(qkv, nh, nkv, hd, positions, inv_freq, interleaved, qk_norm, eps, temperature, seq, table, k16, v16, page, write,
                            q_norm_weight=qw, k_norm_weight=kw, norm_first=first, norm_dim=dim, rot_mul=mul, values_are_keys=keys_as_values)
        assert ((q.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 2.0 ** -20 * want.double().abs().max()).all()
        if write:
            at, row = table[seq.long(), (positions // page).long()].long(), (positions % page).long()
            n = positions.numel()
            cu = torch.arange(n + 1, dtype=torch.int32, device=qkv.device)
            k4, v4, _ = ops.expand_pages_4bit(kv_pages, hd, table[seq.long()].contiguous(), cu, positions, positions.tolist(), [1] * n, window=1)
            index = torch.arange(n, device=qkv.device)
            for got, full in ((k4, k16), (v4, v16)):
                a, b = got[index, :, row].double(), full[at, :, row].double()
                groups = b.unflatten(-1, (-1, GROUP))
                step = ((groups.amax(-1) - groups.amin(-1)) / 15).repeat_interleave(GROUP, -1)
                # half a step, the scale's rounding at 15 of them, the key's own rounding (now and then the other way), the value's
                assert ((a - b).abs() <= step * (0.5 + 15 * 2.0 ** -8) * (1 + 2.0 ** -6) + 2.0 ** -6 * b.abs()).all()
        seen["appends"] += 1
        return q

    def checked_attend(q, kv_pages, table, ctx, nh, nkv, hd, chunk, sliding, scale, sink=False, softcap=0.0, slopes=None, sink_values=None,
                       keep=0):
        o = attend(q, kv_pages, table, ctx, nh, nkv, hd, chunk, sliding, scale, sink=sink, softcap=softcap, slopes=slopes,
                   sink_values=sink_values, keep=keep)
        assert not o.isnan().any()
        sinks = sink_values if sink_values is not None else torch.zeros(nh, device=q.device) if sink else None
        for s, (start, n) in enumerate(zip(ctx.start_pos, ctx.n_new)):
            at = slice(int(ctx.cu_seqlens[s]), int(ctx.cu_seqlens[s + 1]))
            length = start + n
            page = kv_pages.shape[2] * 4 // (5 * hd)
            mask = visible(ctx.positions[at], length, chunk, sliding, keep)
            cu = torch.tensor([0, n], dtype=torch.int32, device=q.device)
            k, v, new = ops.expand_pages_4bit(kv_pages, hd, table[s: s + 1], cu, ctx.positions[at].contiguous(), [start], [n], chunk, sliding, keep)
            rows = new[0, torch.arange(length, device=q.device) // page].long().clamp(min=0)
            offset = torch.arange(length, device=q.device) % page
            k, v = k[rows, :, offset].double(), v[rows, :, offset].double()
            hidden = ~mask.any(0)
            k[hidden], v[hidden] = 0.0, 0.0
            if softcap or slopes is not None:
                continue
            want, size = attention(q[at], k, v, mask, scale, sinks)
            # what the reference takes are the cached rows rounded to bfloat16 (2^-8 of a key: off scores by that times scale sum |q| |k|, twice
            # that a weight; 2^-8 of a value), and the kernels round weights and result likewise (values by parts up to 3 of the largest)
            off = 2.0 ** -8 * scale * torch.einsum("nhd,thd->nht", q[at].double().abs(), k.abs().repeat_interleave(nh // nkv, 1))
            off = off.masked_fill(~mask.unsqueeze(1), 0).amax(-1, keepdim=True)
            tol = 2 * off * (1 + off) * size + 2.0 ** -8 * (2 * size + 3 * v.abs().amax() + 3 * want.abs())
            assert ((o[at].double() - want).abs() <= tol).all()
        seen["attends"] += 1
        return o

    monkeypatch.setattr(ops, "qkv_post_4bit", checked_post)
    monkeypatch.setattr(parts, "attend_over_four_bit_pages", checked_attend)


def _drive(eng, toks, other):
    from hi_b200.engine.core import StepEntry

    out = [eng.step([StepEntry("a", toks[:70], [69])])]
    out.append(eng.step([StepEntry("a", toks[70:75], [4]), StepEntry("b", other[:3], [2])]))
    out.append(eng.step([StepEntry("a", toks[75:76], [0]), StepEntry("b", other[3:40], [36]), StepEntry("c", toks[:1], [0])]))
    for i in range(20):
        out.append(eng.step([StepEntry("a", [toks[76 + i]], [0]), StepEntry("b", [other[40 + i]], [0]), StepEntry("c", [toks[1 + i]], [0])]))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("which", ["llama4", "fidatar", "bezasun"])
def test_every_step_against_the_cached_rows(which, page, tmp_path, monkeypatch):
    """Prompts, portions of a few tokens, mixed steps and decoding over pages that are poisoned when they are given back."""
    from hi_b200.engine.core import Engine

    if which == "llama4":
        cfg, mdir = TINY_A, h.make_model(str(tmp_path / "m"), TINY_A, seed=5)
    elif which == "fidatar":
        cfg = fidatar_configs.config(131, 64, 1e-5, [
            fidatar_configs.attention(4, 2, 24, 16, 0.3, chunk=32, rot=fidatar_configs.rot(16, 10000.0), mlp=fidatar_configs.dense(64)),
            fidatar_configs.mlstm(2, 16, 16, 12.0), fidatar_configs.attention(6, 3, 16, 16, 0.25)])
        mdir = str(tmp_path / "m")
        fidatar_configs.write_model(mdir, cfg, 4)
    else:
        cfg = bezasun_configs.config(131, 64, 1e-5, [bezasun_configs.attention(4, 2, 16, 16, 0.25, softcap=20.0, mlp=None)])
        mdir = str(tmp_path / "m")
        bezasun_configs.write_model(mdir, cfg, 4)
    seen = {"appends": 0, "attends": 0}
    _watch(monkeypatch, seen)
    eng = Engine.from_dir(mdir, kv_page_size=page, kv_cache_tokens=640, max_active_requests=4, kv_cache_bits=4, debug_poison=True,
                          use_cuda_graphs=False)
    toks, other = ([(7 * i + s) % 128 for i in range(128)] for s in (1, 5))
    for logits in _drive(eng, toks, other):
        assert logits.isfinite().all()
    layers = sum(1 for cs in eng.model.cache_specs.values() if cs is not None and cs.paged)
    assert layers > 0 and seen["appends"] == seen["attends"] == 23 * layers


@pytest.mark.gpu
def test_captured_steps_are_the_eager_ones(tmp_path):
    from hi_b200.engine.core import Engine

    mdir = h.make_model(str(tmp_path / "m"), TINY_A, seed=6)
    toks, other = ([(5 * i + s) % 200 for i in range(128)] for s in (1, 9))
    runs = []
    for graphs in (True, False):
        eng = Engine.from_dir(mdir, kv_page_size=16, kv_cache_tokens=640, max_active_requests=4, kv_cache_bits=4, weight_bits=4,
                              use_cuda_graphs=graphs, graph_context_bucket=128)
        runs.append(_drive(eng, toks, other))
        assert bool(eng._graphs) == graphs
    for a, b in zip(*runs):
        assert h.rel_err(a, b.cpu()) <= h.TOL_BF16      # (the cut of the keys goes by the bucket in the one, by the longest in the other)


@pytest.mark.gpu
def test_generate_and_command(tmp_path, capsys):
    import json

    import hi_b200
    from hi_b200.cli import main

    mdir = h.make_model(str(tmp_path / "m"), TINY_A, seed=7)
    outs = hi_b200.generate(mdir, [[1, 2, 3], list(range(40))], hi_b200.SamplingParams(max_tokens=6), kv_cache_bits=4, weight_bits=4,
                            kv_cache_tokens=512)
    assert [len(o.token_ids) for o in outs] == [6, 6] or any(o.finish_reason == "stop" for o in outs)
    assert main(["run", mdir, "--tokens", "1,2,3", "--max-tokens", "4", "--kv-cache-bits", "4", "--weight-bits", "4", "--weight-group", "32"]) == 0
    assert len(json.loads(capsys.readouterr().out)["top_logits"]) == 5


def test_a_pool_sized_from_memory_holds_more_tokens():
    from hi_b200.cache.device import pool_tokens_for_budget
    from hi_b200.config.registry import lookup
    from hi_b200.parts.model import Model

    cfg = dict(TINY_A, head_dim=128, attention_chunk_size=1 << 20)
    arch = lookup(cfg)
    spec = arch.build_spec(arch.parse_config(cfg, None))
    few, many = (pool_tokens_for_budget(Model(spec, BF16, "cpu", cache_bits=b).cache_specs, 2, 1 << 26, 64, 2) for b in (16, 4))
    assert sum(many) >= 3.1 * sum(few)
