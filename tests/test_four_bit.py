"""Products with 4-bit weights, the append to a 4-bit cache and attention over it, against plain forms in float64."""
import pytest
import torch

from plain_four_bit import attention, quantise, unpack_weight, values, visible, weight_values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _weight(m, k, group, g):
    from hi_b200.kernels import ops

    codes = torch.randint(0, 16, (m, k), device=DEV, generator=g).to(torch.uint8)
    scales = ((0.5 + torch.rand(m, k // group, device=DEV, generator=g)) * 0.2 * k ** -0.5).to(BF16)
    return ops.pack_weight(codes, scales), codes, scales


def _check_linear(got, x, codes, scales, bias=None):
    """Up to 16 tokens: products of whole numbers with x are exact; what is rounded: float32 sums (the tensor cores drop what lies 2^-23 under the
    largest term, up to 9 times a group, then a few dozen additions: 2^-18 of the sum of all magnitudes, the eights' among them) and
    the result. More tokens: each weight is rounded to bfloat16, 2^-8 of every product, and the float32 sums as before."""
    want = x.double() @ weight_values(codes, scales).t()
    size = x.double().abs() @ ((codes.double() + 8) * scales.double().repeat_interleave(codes.shape[1] // scales.shape[1], 1)).t()
    if bias is not None:
        want = want + bias.double()
    tol = 2.0 ** -18 * size
    if x.shape[0] > 16:
        tol = tol + 2.0 ** -8 * (x.double().abs() @ weight_values(codes, scales).abs().t())
    if got.dtype == BF16:
        tol = tol + 2.0 ** -8 * want.abs()
    else:
        tol = tol + 2.0 ** -24 * want.abs()
    assert got.shape == want.shape and ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("m,k,group", [(1, 32, 32), (15, 64, 64), (16, 128, 128), (17, 2048, 64), (100, 2080, 32), (2400, 384, 128),
                                       (64, 13312, 128), (40, 6976, 64)])
@pytest.mark.parametrize("tokens", [1, 7, 8, 9, 16, 17, 40])
@pytest.mark.parametrize("out_dtype", [torch.float32, BF16])
def test_linear(m, k, group, tokens, out_dtype):
    from hi_b200.parts.linear import linear

    g = _gen(m + k + tokens)
    w, codes, scales = _weight(m, k, group, g)
    wide = torch.randn(tokens, k + 24, device=DEV, generator=g).to(BF16)
    x = wide[:, 8: 8 + k]
    bias = torch.randn(m, device=DEV, generator=g).to(BF16)
    from hi_b200.kernels import ops

    _check_linear(linear(x, w, out_dtype=out_dtype), x, codes, scales)
    _check_linear(linear(x, w, out_dtype=out_dtype, bias=bias), x, codes, scales, bias)
    ops.check_tc_status()


@pytest.mark.parametrize("m,k,group", [(16, 32, 32), (129, 640, 128), (300, 2112, 64), (5000, 1056, 32), (9700, 256, 128), (19200, 128, 64)])
@pytest.mark.parametrize("tokens", [17, 64, 65, 128, 129, 200, 256, 257, 600])
def test_linear_of_many_tokens(m, k, group, tokens):
    """Row tiles of 128 and of a pair's 256 that are not full, one block a tile and clusters that share K, tiles of 64, 128 and up to 256
    tokens, more tiles than blocks; against the product with the rounded weights too, which leaves float32 sums."""
    from hi_b200.kernels import ops
    from hi_b200.parts.linear import linear

    g = _gen(m + k + tokens)
    w, codes, scales = _weight(m, k, group, g)
    wide = torch.randn(tokens, k + 8, device=DEV, generator=g).to(BF16)
    x = wide[:, :k]
    bias = torch.randn(m, device=DEV, generator=g).to(BF16)
    got = linear(x, w, out_dtype=torch.float32, bias=bias)
    ops.check_tc_status()
    rounded = weight_values(codes, scales).to(BF16).double()
    want, size = x.double() @ rounded.t() + bias.double(), x.double().abs() @ rounded.abs().t()
    assert ((got.double() - want).abs() <= 2.0 ** -18 * size + 2.0 ** -24 * want.abs()).all()
    got16 = linear(x, w, bias=bias)
    assert torch.equal(got16, got.to(BF16)) and torch.equal(linear(x.contiguous(), w, bias=bias), got16)
    ops.check_tc_status()


@pytest.mark.parametrize("m,k,group", [(128, 8192, 128), (600, 2048, 64), (1024, 4000, 32), (2048, 2048, 64), (5120, 1024, 128), (4090, 1792, 32)])
@pytest.mark.parametrize("tokens", [17, 100, 200, 384, 530])
def test_linear_of_few_tiles(m, k, group, tokens):
    """Two to eight blocks that share K, with one tile of tokens and with several, shares of unlike length, the last ones short."""
    from hi_b200.kernels import ops

    g = _gen(m + k + tokens + 1)
    w, codes, scales = _weight(m, k, group, g)
    x = torch.randn(tokens, k, device=DEV, generator=g).to(BF16)
    bias = torch.randn(m, device=DEV, generator=g).to(BF16)
    got = ops.four_bit_linear(x, w, torch.float32, bias)
    rounded = weight_values(codes, scales).to(BF16).double()
    want, size = x.double() @ rounded.t() + bias.double(), x.double().abs() @ rounded.abs().t()
    assert ((got.double() - want).abs() <= 2.0 ** -18 * size + 2.0 ** -24 * want.abs()).all()
    ops.check_tc_status()


@pytest.mark.parametrize("m,k,group", [(33, 50048, 32), (20, 26112, 128), (1200, 8192, 64), (3000, 2048, 128), (16, 384, 64)])
@pytest.mark.parametrize("tokens", [1, 8, 16])
def test_linear_of_blocks_that_share_k(m, k, group, tokens):
    """One, two and four blocks on a row tile's K, inputs that shared memory holds and such that come in parts, several row tiles a block."""
    from hi_b200.kernels import ops

    g = _gen(m + k + tokens + 2)
    w, codes, scales = _weight(m, k, group, g)
    x = torch.randn(tokens, k, device=DEV, generator=g).to(BF16)
    bias = torch.randn(m, device=DEV, generator=g).to(BF16)
    for kind in (torch.float32, BF16):
        _check_linear(ops.four_bit_linear(x, w, kind, bias), x, codes, scales, bias)


def test_linear_edges():
    """No tokens; rows that start anywhere; large and small inputs; a scale of zero and one that is not finite."""
    from hi_b200.kernels import ops
    from hi_b200.parts.linear import linear

    g = _gen(5)
    w, codes, scales = _weight(33, 256, 32, g)
    x = torch.randn(4, 256, device=DEV, generator=g).to(BF16)
    assert linear(x[:0], w).shape == (0, 33)
    flat = torch.randn(4 * 256 + 1, device=DEV, generator=g).to(BF16)
    for a in (flat[1:].view(4, 256), x.t().contiguous().t(), x[:, :].expand(4, 256), x[::2], x[:1].expand(5, 256)):
        _check_linear(linear(a, w, out_dtype=torch.float32), a, codes, scales)
    for size in (2.0 ** 60, 2.0 ** -40):
        _check_linear(linear(x * size, w, out_dtype=torch.float32), x * size, codes, scales)
    scales[3, 2], scales[4, 1] = 0.0, float("nan")
    y = linear(x, ops.pack_weight(codes, scales))
    assert y[:, 4].isnan().all() and int(y.isnan().sum()) == 4
    keep = [r for r in range(33) if r != 4]
    _check_linear(y[:, keep], x, codes[keep], scales[keep])


def test_linear_refusals():
    from hi_b200.kernels import ops
    from hi_b200.parts.linear import linear

    w, _, _ = _weight(16, 64, 64, _gen(1))
    x = torch.zeros(2, 64, dtype=BF16, device=DEV)
    for bad in (x[:, :32], x.float(), x[0], x.requires_grad_(False).half()):
        with pytest.raises(ops.KernelError):
            ops.four_bit_linear(bad, w)
    for kw in (dict(out_dtype=torch.float16), dict(bias=torch.zeros(15, dtype=BF16, device=DEV)), dict(bias=torch.zeros(16, device=DEV))):
        with pytest.raises(ops.KernelError):
            ops.four_bit_linear(x, w, **kw)
    with pytest.raises(ops.KernelError):
        linear(torch.zeros(2, 64, dtype=BF16, device=DEV, requires_grad=True), w)


# --------------------------------------------------------------------------- the cache
class Step:
    """Requests (new tokens, cached tokens) with rows of their own in a 4-bit pool; what no token wrote is NaN."""

    def __init__(self, portions, nh, nkv, hd, page, seed=0, spare=2):
        from hi_b200.kernels import ops
        from hi_b200.parts.context import StepContext

        g = _gen(seed)
        n_new, start = [n for n, _c in portions], [c for _n, c in portions]
        cu = [0]
        for n in n_new:
            cu.append(cu[-1] + n)
        need = [-(-(n + c) // page) for n, c in portions]
        order = torch.randperm(sum(need) + spare, device=DEV, generator=g).to(torch.int32)
        self.table = torch.full((len(portions), max(need + [1]) + 1), -1, dtype=torch.int32, device=DEV)
        at = 0
        for s, k in enumerate(need):
            self.table[s, :k] = order[at: at + k]
            at += k
        self.pages = torch.full((sum(need) + spare, nkv, ops.four_bit_page_bytes(page, hd)), 255, dtype=torch.uint8, device=DEV)
        self.nh, self.nkv, self.hd, self.page, self.portions, self.cu = nh, nkv, hd, page, portions, cu
        self.positions = torch.cat([torch.arange(c, c + n) for n, c in portions]).to(torch.int32).to(DEV)
        self.seq = torch.repeat_interleave(torch.arange(len(portions)), torch.tensor(n_new)).to(torch.int32).to(DEV)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        self.ctx = StepContext(n_tokens=cu[-1], n_seqs=len(portions), tokens=self.positions, positions=self.positions,
                               seq_of_token=self.seq, cu_seqlens=i32(cu), slots=i32(list(range(len(portions)))), start_pos=start,
                               n_new=n_new, slot_ids=list(range(len(portions))), page_size=page,
                               max_context=max(n + c for n, c in portions))
        singles = [i for i, n in enumerate(n_new) if n == 1]
        if singles and len(singles) < len(n_new):
            self.ctx.decode_rows = torch.tensor([cu[i] for i in singles], dtype=torch.int64, device=DEV)
            self.ctx.decode_max_context = max(start[i] + 1 for i in singles)
        self.q = torch.randn(cu[-1], nh, hd, device=DEV, generator=g).to(BF16)
        self.k, self.v = [], []
        for s, (n, c) in enumerate(portions):
            k = torch.randn(n + c, nkv, hd, device=DEV, generator=g) * torch.exp(0.5 * torch.randn(nkv, hd, device=DEV, generator=g)) + 0.3
            v = torch.randn(n + c, nkv, hd, device=DEV, generator=g)
            self.k.append(k.to(BF16))
            self.v.append(v.to(BF16))

    def fill(self):
        for s, (n, c) in enumerate(self.portions):
            rows = torch.cat([self.k[s].flatten(1), self.k[s].flatten(1), self.v[s].flatten(1)], 1).contiguous()
            self.append(rows, self.nkv, torch.arange(n + c, dtype=torch.int32, device=DEV),
                        torch.full((n + c,), s, dtype=torch.int32, device=DEV))
        return self

    def append(self, qkv, nh, positions, seq, **kw):
        from hi_b200.kernels import ops

        return ops.qkv_post_4bit(qkv, nh, self.nkv, self.hd, positions, None, False, False, 1e-6, None, seq, self.table, self.pages, **kw)

    def expected(self, s, **mask):
        k, v = values(quantise(self.k[s])), values(quantise(self.v[s]))
        a, b = self.cu[s], self.cu[s + 1]
        return self.q[a:b], k, v, visible(self.positions[a:b], k.shape[0], **mask)


@pytest.mark.parametrize("hd,page", [(128, 64), (64, 64), (128, 16), (64, 32), (128, 192)])
def test_append_and_expand_bit_by_bit(hd, page):
    """Codes, scales and lows as float32 arithmetic gives them; rows beside the new ones stay; the spans of pages and their table."""
    from hi_b200.kernels import ops

    step = Step([(37, 0), (1, 200), (70, 3), (2, 63)], 3, 3, hd, page, seed=hd + page)
    step.k[2][5, 1, :32] = 0.25                      # a group of one value
    step.v[0][7, 2, 32:64] = torch.arange(32, device=DEV).to(BF16)     # exact steps, ties among the codes of a rounded scale
    step.k[3][64, 0, 3] = float("inf")
    step.v[3][64, 0, 40] = float("nan")
    step.fill()
    ctx = step.ctx
    for chunk, window, keep, skip in ((0, 0, 0, False), (64, 0, 0, False), (0, 20, 0, True), (0, 20, 5, False), (0, 1, 0, False)):
        k, v, table = ops.expand_pages_4bit(step.pages, hd, step.table, ctx.cu_seqlens, step.positions, ctx.start_pos, ctx.n_new,
                                            chunk, window, keep, skip)
        at = 0
        for s, (n, c) in enumerate(step.portions):
            if skip and n == 1:
                continue
            low = c // chunk * chunk if chunk else max(0, c - window + 1) if window and not keep else 0
            first, last = low // page, (c + n - 1) // page
            for pool, rows in ((k, step.k[s]), (v, step.v[s])):
                want = values(quantise(rows), torch.float32).to(BF16)[first * page:]
                got = pool[at: at + last - first + 1].transpose(1, 2).reshape(-1, 3, hd)[: want.shape[0]]
                assert torch.equal(got.view(torch.int16)[~want.isnan()], want.view(torch.int16)[~want.isnan()])
                assert torch.equal(got.isnan(), want.isnan())
            assert table[s, first: last + 1].tolist() == list(range(at, at + last - first + 1))
            at += last - first + 1
        assert k.shape[0] == at


@pytest.mark.parametrize("hd,nh,nkv", [(128, 5, 2), (64, 6, 3)])
@pytest.mark.parametrize("form", ["rope", "rope_interleaved", "partial", "norm_after", "norm_first", "keys_as_values", "no_write"])
def test_append_encodes_as_the_bfloat16_cache_does(hd, nh, nkv, form):
    from hi_b200.kernels import ops

    g = _gen(hd + len(form))
    n, page = 45, 64
    one = form == "keys_as_values"
    qkv = torch.randn(n, (nh + (1 if one else 2) * nkv) * hd, device=DEV, generator=g).to(BF16)
    positions = torch.cat([torch.arange(30, 60), torch.arange(5000, 5015)]).to(torch.int32).to(DEV)
    seq = torch.tensor([0] * 30 + [1] * 15, dtype=torch.int32, device=DEV)
    table = torch.full((2, 80), -1, dtype=torch.int32, device=DEV)
    table[0, 0], table[1, 78] = 1, 0
    inv = 500000.0 ** (-torch.arange(hd // 2, device=DEV, dtype=torch.float32) / (hd // 2))
    kw = {}
    norm, dim, inter, freq = False, 0, form == "rope_interleaved", inv
    if form == "partial":
        freq = inv[: hd // 2 - 3].contiguous()
        kw = dict(rot_mul=1.25)
    if form == "norm_after":
        norm = True
    if form in ("norm_first", "keys_as_values"):
        norm = True
        kw = dict(norm_first=True, q_norm_weight=torch.rand(hd, device=DEV, generator=g), k_norm_weight=torch.rand(hd, device=DEV, generator=g))
    if one:
        kw["values_are_keys"] = True
    k16, v16 = (torch.zeros(2, nkv, page, hd, dtype=BF16, device=DEV) for _ in range(2))
    want = ops.qkv_post(qkv, nh, nkv, hd, positions, freq, inter, norm, 1e-5, (512.0, 0.1), seq, table, k16, v16, page, True, norm_dim=dim, **kw)
    pages = torch.zeros(2, nkv, ops.four_bit_page_bytes(page, hd), dtype=torch.uint8, device=DEV)
    got = ops.qkv_post_4bit(qkv, nh, nkv, hd, positions, freq, inter, norm, 1e-5, (512.0, 0.1), seq, table, pages,
                            write_kv=form != "no_write", **kw)
    # the same formulas: float32, then one rounding to bfloat16 (2^-8), which falls the other way now and then
    assert ((got.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 1e-6).all()
    if form == "no_write":
        assert not pages.any()
        return
    cu = torch.tensor([0, 30, 45], dtype=torch.int32, device=DEV)
    k, v, _ = ops.expand_pages_4bit(pages, hd, table, cu, positions, [30, 5000], [30, 15], window=1)
    for pool, full in ((k, k16), (v, v16)):
        for mine, src, rows in ((0, 1, slice(30, 60)), (1, 0, slice(5000 % 64, 5000 % 64 + 15))):
            a, b = pool[mine][:, rows].double(), full[src][:, rows].double()
            spread = b.unflatten(-1, (-1, 32)).amax(-1) - b.unflatten(-1, (-1, 32)).amin(-1)
            step = (spread / 15).repeat_interleave(32, -1)
            # half a step, the scale's rounding at 15 steps, the key's own rounding and that of the expanded value
            assert ((a - b).abs() <= step * (0.5 + 15 * 2.0 ** -8) * (1 + 2.0 ** -6) + 2.0 ** -6 * b.abs()).all()


DECODE = [
    # heads, kv heads, dim, page, portions (new, cached), mask
    (40, 8, 128, 64, [(1, 0)], {}),
    (40, 8, 128, 64, [(1, 999)], {}),
    (32, 8, 64, 64, [(1, 63), (1, 64), (1, 0), (1, 15), (1, 16), (1, 4000)], {}),
    (8, 8, 128, 16, [(1, 31), (1, 500), (1, 7)], {}),
    (16, 1, 64, 32, [(1, 1000), (1, 33)], {}),
    (17, 1, 128, 64, [(1, 300)], {}),
    (10, 2, 128, 192, [(1, 5000), (1, 191), (1, 192)], {}),
    (16, 4, 128, 64, [(1, 8190), (1, 8192), (1, 100), (1, 9000)], dict(chunk=8192)),
    (16, 4, 64, 32, [(1, 700), (1, 99), (1, 100)], dict(chunk=100)),
    (16, 4, 128, 64, [(1, 3000), (1, 50), (1, 99), (1, 1023)], dict(window=100)),
    (16, 4, 64, 16, [(1, 3000), (1, 2), (1, 130), (1, 64 * 20 - 1)], dict(window=64, keep=3)),
    (16, 4, 128, 64, [(1, 700), (1, 71), (1, 1500)], dict(window=65, keep=130)),
    (16, 4, 128, 64, [(1, 700), (1, 1)], dict(window=1)),
    (8, 2, 128, 64, [(1, 70000)], {}),
]


def _check_rows(step, s, got, mask, scale, sink, decoded):
    q, k, v, seen = step.expected(s, **mask)
    want, size = attention(q, k, v, seen, scale, sink)
    if decoded:
        # weights are rounded to bfloat16 (2^-8) times the scale, before codes less eight, and bare, before the group's middle and in the
        # sum of weights; scores are off by float32 sums only (2^-13 of the weights covers |score| up to 500); the result is rounded
        codes, t, low = quantise(step.v[s])
        t, low = t.double().unsqueeze(-1), low.double().unsqueeze(-1)
        grown = (t * (codes.double().unflatten(-1, (-1, 32)) - 8).abs() + (low + 8 * t).abs()).flatten(-2)
        _, size = attention(q, k, grown, seen, scale, sink)
        tol = 2.0 ** -8 * (size + 2 * want.abs()) + 2.0 ** -13 * size
    else:
        # keys, values and weights in float16 (2^-11 each; the queries are exact in it but for parts 2^-25 of a key's and a query's largest):
        # a score is off by up to 2^-11 scale sum |q| |k|, and twice that moves a weight against its sum; the result is rounded
        per = q.shape[1] // k.shape[1]
        off = 2.0 ** -10.5 * scale * torch.einsum("nhd,thd->nht", q.double().abs(), k.abs().repeat_interleave(per, 1))
        off = off.masked_fill(~seen.unsqueeze(1), 0).amax(-1, keepdim=True)
        tol = (2 * off * (1 + off) + 3 * 2.0 ** -11) * size + 2.0 ** -11 * want.abs() + 2.0 ** -8 * want.abs() + 2.0 ** -20 * size.amax()
    diff = (got[step.cu[s]: step.cu[s + 1]].double() - want).abs()
    assert (diff <= tol).all(), (s, float((diff / tol).max()))


def _check_decode(step, got, mask, scale, sink=None):
    for s in range(len(step.portions)):
        _check_rows(step, s, got, mask, scale, sink, True)


@pytest.mark.parametrize("case", DECODE, ids=lambda c: f"{c[0]}on{c[1]}x{c[2]}p{c[3]}n{len(c[4])}" + "".join(f"_{k}{v}" for k, v in c[5].items()))
def test_decode(case):
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages

    nh, nkv, hd, page, portions, mask = case
    step = Step(portions, nh, nkv, hd, page, seed=nh + hd).fill()
    chunk, window, keep = mask.get("chunk", 0), mask.get("window", 0), mask.get("keep", 0)
    scale = hd ** -0.5
    got = attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, nh, nkv, hd, chunk, window, scale, keep=keep)
    ops.check_tc_status()
    _check_decode(step, got, mask, scale)
    sinks = torch.randn(nh, device=DEV, generator=_gen(3)) * 3
    got = attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, nh, nkv, hd, chunk, window, scale, sink=True, keep=keep)
    _check_decode(step, got, mask, scale, torch.zeros(nh, device=DEV))
    got = attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, nh, nkv, hd, chunk, window, scale, sink_values=sinks, keep=keep)
    _check_decode(step, got, mask, scale, sinks)


@pytest.mark.parametrize("splits", [1, 2, 5, 33])
def test_decode_in_any_cut(splits, monkeypatch):
    """The same keys in one split and in many, also more than there are tiles for."""
    from hi_b200.kernels import ops

    step = Step([(1, 2100), (1, 64), (1, 700)], 16, 4, 128, 64, seed=splits).fill()
    monkeypatch.setattr(ops, "_four_bit_splits", lambda tiles, groups, hd: (-(-tiles // splits), splits))
    got = ops.decode_attention_4bit(step.q, step.pages, step.table, step.seq, step.positions, 0, 0, 0.1, 2101)
    ops.check_tc_status()
    _check_decode(step, got, {}, 0.1)


def test_decode_of_some_rows():
    """Tokens of a step decoded where they lie: other rows of the output stay, a row outside the step is left out and found."""
    from hi_b200.kernels import ops

    step = Step([(1, 300), (1, 4), (1, 90), (1, 64)], 8, 2, 64, 64, seed=9).fill()
    out = torch.full_like(step.q, 7.0)
    rows = torch.tensor([3, 1], dtype=torch.int64, device=DEV)
    ops.decode_attention_4bit(step.q, step.pages, step.table, step.seq, step.positions, 0, 0, 0.125, 301, rows=rows, out=out)
    assert (out[0] == 7).all() and (out[2] == 7).all()
    whole = ops.decode_attention_4bit(step.q, step.pages, step.table, step.seq, step.positions, 0, 0, 0.125, 301)
    ops.check_tc_status()
    assert torch.equal(out[1], whole[1]) and torch.equal(out[3], whole[3])
    ops.decode_attention_4bit(step.q, step.pages, step.table, step.seq, step.positions, 0, 0, 0.125, 301,
                              rows=torch.tensor([0, 4], dtype=torch.int64, device=DEV), out=out)
    with pytest.raises(ops.KernelError, match="row outside"):
        ops.check_tc_status()
    assert torch.equal(out[0], whole[0])
    none = ops.decode_attention_4bit(step.q[:0], step.pages, step.table, step.seq[:0], step.positions[:0], 0, 0, 0.125, 1)
    assert none.shape == (0, 8, 64)
    # a token at no position (padding) reads nothing
    step.positions[2] = -1
    padded = ops.decode_attention_4bit(step.q, step.pages, step.table, step.seq, step.positions, 0, 0, 0.125, 301)
    assert not padded[2].any() and torch.equal(padded[0], whole[0])
    # a position behind the pages that the table names: the keys that are there
    short = step.table[:, :2].contiguous()
    clipped = torch.tensor([127, 4, -1, 64], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.decode_attention_4bit(step.q, step.pages, short, step.seq, step.positions, 0, 0, 0.125, 301),
                       ops.decode_attention_4bit(step.q, step.pages, short, step.seq, clipped, 0, 0, 0.125, 301))
    assert not ops.decode_attention_4bit(step.q, step.pages, short, step.seq, step.positions, 0, 50, 0.125, 301)[0].any()


def test_a_key_that_is_not_finite_shows():
    from hi_b200.kernels import ops

    step = Step([(1, 130), (1, 0), (1, 130)], 8, 2, 128, 64, seed=4)
    step.k[0][70, 1, 3] = float("nan")
    step.v[1][0, 0, 100] = float("inf")
    step.fill()
    got = ops.decode_attention_4bit(step.q, step.pages, step.table, step.seq, step.positions, 0, 0, 0.1, 131)
    assert got[0, 4:].isnan().all() and not got[0, :4].isnan().any()
    assert got[1, :4, 96:].isnan().all() and not got[1, :4, :96].isnan().any() and not got[1, 4:].isnan().any()
    assert not got[2].isnan().any()


PORTIONS = [
    (40, 8, 128, 64, [(130, 0), (1, 500), (64, 700), (1, 3), (5, 61)], {}),
    (16, 4, 64, 64, [(3, 100), (1, 64), (2, 0)], {}),
    (16, 4, 128, 64, [(200, 1000), (1, 2000)], dict(window=100)),
    (16, 4, 128, 64, [(200, 1000), (1, 2000)], dict(window=100, keep=70)),
    (16, 4, 64, 32, [(100, 450), (1, 513), (1, 511)], dict(chunk=256)),
    (8, 8, 128, 16, [(70, 20), (1, 99)], {}),
    (16, 4, 128, 64, [(14, 200), (9, 0), (1, 5)], dict(window=30)),
    (48, 4, 64, 64, [(9, 300), (12, 90), (1, 64)], {}),
]


@pytest.mark.parametrize("case", PORTIONS, ids=lambda c: f"{c[0]}on{c[1]}x{c[2]}p{c[3]}" + "".join(f"_{k}{v}" for k, v in c[5].items()))
def test_portions(case):
    """Portions beside single tokens: the former over the expanded pages, the latter, and steps of a few tokens a request, as they are."""
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import FOUR_BIT_DECODED, attend_over_four_bit_pages

    nh, nkv, hd, page, portions, mask = case
    step = Step(portions, nh, nkv, hd, page, seed=nh + page).fill()
    scale = hd ** -0.5
    few = max(n for n, _c in portions) * -(-(nh // nkv) // 8) <= FOUR_BIT_DECODED
    for sink in (None, torch.randn(nh, device=DEV, generator=_gen(3))):
        got = attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, nh, nkv, hd, mask.get("chunk", 0), mask.get("window", 0),
                                         scale, sink_values=sink, keep=mask.get("keep", 0))
        ops.check_tc_status()
        for s, (n, _c) in enumerate(portions):
            _check_rows(step, s, got, mask, scale, sink, few or n == 1)


@pytest.mark.parametrize("k_size,v_size,q_size", [(2.0 ** 30, 2.0 ** -40, 2.0 ** -30), (2.0 ** -20, 2.0 ** 60, 2.0 ** 18), (1.0, 2.0 ** -20, 1.0)])
def test_portions_of_any_size(k_size, v_size, q_size):
    """Keys and values that float16 does not hold as they are."""
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages

    step = Step([(40, 100), (150, 0), (1, 70)], 8, 2, 128, 64, seed=12)
    step.k, step.v, step.q = [k * k_size for k in step.k], [v * v_size for v in step.v], step.q * q_size
    step.v[0][:, 1] *= 2.0 ** -10                # one head's values much smaller than the other's
    step.fill()
    got = attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, 8, 2, 128, 0, 0, 0.09)
    ops.check_tc_status()
    for s in range(3):
        _check_rows(step, s, got, {}, 0.09, None, s == 2)


def test_reshaped_scores_go_over_bfloat16_pages():
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages, attend_over_pages

    step = Step([(40, 100), (1, 70), (1, 900)], 8, 2, 64, 64, seed=13).fill()
    slopes = torch.rand(8, device=DEV, generator=_gen(1)) * 0.01
    ctx = step.ctx
    k, v, table = ops.expand_pages_4bit(step.pages, 64, step.table, ctx.cu_seqlens, step.positions, ctx.start_pos, ctx.n_new)
    want = attend_over_pages(step.q, k, v, table, ctx, 8, 2, 64, 0, 0, 0.125, softcap=20.0, slopes=slopes)
    got = attend_over_four_bit_pages(step.q, step.pages, step.table, ctx, 8, 2, 64, 0, 0, 0.125, softcap=20.0, slopes=slopes)
    ops.check_tc_status()
    assert torch.equal(got, want) and not got.isnan().any()


def test_cache_refusals():
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages

    step = Step([(1, 70), (1, 9)], 8, 2, 64, 64).fill()
    q, pages, table, seq, pos = step.q, step.pages, step.table, step.seq, step.positions
    call = lambda q=q, pages=pages, table=table, seq=seq, pos=pos, **kw: \
        ops.decode_attention_4bit(q, pages, table, seq, pos, 0, 0, 0.1, 71, **kw)
    for kw in (dict(q=q.float()), dict(q=q[0]), dict(pages=pages.to(torch.int8)), dict(pages=pages[:, :, :-80]), dict(pages=pages[0]),
               dict(seq=seq[:1]), dict(pos=pos.long()), dict(table=table[0]), dict(q=q[:, :7].contiguous()), dict(out=torch.empty_like(q)),
               dict(rows=torch.zeros(1, dtype=torch.int64, device=DEV)), dict(rows=torch.zeros(1, dtype=torch.int32, device=DEV), out=torch.empty_like(q)),
               dict(sink_values=torch.zeros(7, device=DEV)), dict(q=torch.zeros(2, 8, 96, dtype=BF16, device=DEV))):
        with pytest.raises(ops.KernelError):
            call(**kw)
    odd = torch.empty(q.numel() + 4, dtype=BF16, device=DEV)[4:].view_as(q)          # rows that start between 16 bytes
    for kw in (dict(q=odd), dict(rows=torch.zeros(1, dtype=torch.int64, device=DEV), out=odd)):
        with pytest.raises(ops.KernelError, match="16 bytes"):
            call(**kw)
    with pytest.raises(ValueError):
        attend_over_four_bit_pages(q, pages, table, step.ctx, 4, 2, 64, 0, 0, 0.1)
    qkv = torch.zeros(2, 12 * 64, dtype=BF16, device=DEV)
    post = lambda qkv=qkv, hd=64, freq=None, temp=None, **kw: \
        ops.qkv_post_4bit(qkv, 8, 2, hd, pos, freq, False, False, 1e-6, temp, seq, table, pages, **kw)
    for kw in (dict(qkv=qkv.float()), dict(qkv=qkv[:, :-64].contiguous()), dict(hd=128), dict(freq=torch.zeros(33, device=DEV)),
               dict(temp=(0.0, 0.1)), dict(norm_dim=65), dict(q_norm_weight=torch.zeros(63, device=DEV))):
        with pytest.raises(ops.KernelError):
            post(**kw)
    cu = step.ctx.cu_seqlens
    for args in ((table, cu, pos, [70], [1, 1]), (table, cu, pos, [70, 64 * 3], [1, 1]), (table, cu[:2], pos, [70, 9], [1, 1]),
                 (table[:1], cu, pos, [70, 9], [1, 1]), (table.long(), cu, pos, [70, 9], [1, 1])):
        with pytest.raises(ops.KernelError):
            ops.expand_pages_4bit(pages, 64, *args)


def test_captured_and_on_another_stream():
    """Projection, append, attention and projection as a decode step runs them: captured, replayed with other contents, on a side stream."""
    from hi_b200.kernels import ops
    from hi_b200.parts.linear import linear

    nh, nkv, hd, width = 16, 4, 128, 512
    step = Step([(1, 900), (1, 63), (1, 0)], nh, nkv, hd, 64, seed=2).fill()
    g = _gen(8)
    w_in, _, _ = _weight((nh + 2 * nkv) * hd, width, 64, g)
    w_out, _, _ = _weight(width, nh * hd, 128, g)
    x = torch.randn(3, width, device=DEV, generator=g).to(BF16)

    def once():
        qkv = linear(x, w_in)
        q = step.append(qkv, nh, step.positions, step.seq)
        o = ops.decode_attention_4bit(q, step.pages, step.table, step.seq, step.positions, 0, 0, hd ** -0.5, 1024)
        return linear(o.view(3, -1), w_out, out_dtype=torch.float32)

    want = once().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    graph.replay()
    assert torch.equal(out, want)
    x.copy_(torch.randn(3, width, device=DEV, generator=g))
    step.positions.copy_(torch.tensor([899, 62, 0], dtype=torch.int32))
    graph.replay()
    got = out.clone()
    assert torch.equal(got, once()) and not torch.equal(got, want)
    ops.check_tc_status()


def test_calls_side_by_side():
    """Products, decode attention and portions on two streams at a time, eager and as two captured graphs, with contents of their own."""
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages
    from hi_b200.parts.linear import linear

    nh, nkv, hd = 16, 4, 128

    def work(seed):
        step = Step([(1, 900 + seed), (70, 200), (1, 0), (300, 40)], nh, nkv, hd, 64, seed=seed).fill()
        single = Step([(1, 1500), (1, 70 + seed)], nh, nkv, hd, 64, seed=seed + 10).fill()
        g = _gen(seed)
        weights = [_weight(m, k, group, g)[0] for m, k, group in ((512, nh * hd, 128), (2000, 512, 32))]
        rows = [torch.randn(n, nh * hd, device=DEV, generator=g).to(BF16) for n in (3, 60, 200)]

        def run():
            out = [linear(linear(x, weights[0]), weights[1]) for x in rows]
            out.append(attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, nh, nkv, hd, 0, 0, 0.09))
            out.append(attend_over_four_bit_pages(single.q, single.pages, single.table, single.ctx, nh, nkv, hd, 0, 0, 0.09))
            return out
        return run

    works = [work(1), work(2)]
    want = [[t.clone() for t in run()] for run in works]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(works[i]())
    torch.cuda.synchronize()
    graphs, outs = [], []
    for run in works:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    ops.check_tc_status()
    for i in (0, 1):
        for result in got[i] + [outs[i]]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[i]))


def test_offsets_that_pass_32_bits():
    """A pool and a weight of more than four gigabytes: pages anywhere in the one, every row tile of the other."""
    from hi_b200.kernels import ops
    from hi_b200.parts.attention import attend_over_four_bit_pages

    step = Step([(1, 700), (130, 20), (1, 63)], 16, 8, 128, 64, seed=21, spare=56000).fill()
    assert step.pages.numel() > 1 << 32 and int(step.table.max()) * step.pages[0].numel() > 1 << 32
    got = attend_over_four_bit_pages(step.q, step.pages, step.table, step.ctx, 16, 8, 128, 0, 0, 0.09)
    for s, (n, _c) in enumerate(step.portions):
        _check_rows(step, s, got, {}, 0.09, None, n == 1)
    ops.check_tc_status()
    del step
    g = _gen(22)
    part, codes, scales = _weight(2048, 65536, 128, g)
    whole = ops.FourBitWeight(part.blocks.repeat(66, 1, 1), (66 * 2048, 65536), 128)
    assert whole.blocks.numel() > 1 << 32
    for n in (3, 40):
        x = torch.randn(n, 65536, device=DEV, generator=g).to(BF16)
        y = ops.four_bit_linear(x, whole, torch.float32).view(n, 66, 2048)
        _check_linear(y[:, 65], x, codes, scales)
        assert torch.equal(y, y[:, :1].expand_as(y))
    ops.check_tc_status()
