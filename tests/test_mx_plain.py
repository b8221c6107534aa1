"""Microscaled 4-bit floats without a GPU: the format of the plain form, packing, refusals."""
import pytest
import torch

import plain_mx
from hi_b200.kernels import ops


def test_the_plain_form_is_the_format():
    """Every code is its own, borders go to the even code, what is above 6 units is 6, exponents follow the largest magnitude."""
    x = torch.zeros(32)
    x[:15] = torch.tensor([0.5, -0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5])
    x[15:19] = torch.tensor([5.0, 7.0, 7.9, -0.2])
    codes, exponents = plain_mx.quantise(x)
    assert exponents.tolist() == [127] and codes[:19].tolist() == [1, 9, 2, 3, 4, 5, 6, 7, 15, 0, 2, 2, 4, 4, 6, 6, 7, 7, 8]
    for top, e in ((4.0, 0), (7.99, 0), (8.0, 1), (3.99, -1), (2.0 ** 127, 125), (2.0 ** -126, -127), (2.0 ** -149, -127), (0.0, -127)):
        assert plain_mx.quantise(torch.full((32,), top))[1].item() == 127 + e, top
    for bad in (float("inf"), float("nan"), -float("inf")):
        x[3] = bad
        assert plain_mx.quantise(x)[1].item() == 255 and plain_mx.held(x).isnan().all()


@pytest.mark.parametrize("shape", [(1, 32), (5, 96), (128, 256), (130, 288), (3, 40, 512), (2, 129, 544)])
def test_packing(shape):
    """Codes two to a byte, scales where the tensor cores look for them."""
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 16, shape, generator=g).to(torch.uint8)
    exps = torch.randint(0, 256, (*shape[:-1], shape[-1] // 32), generator=g).to(torch.uint8)
    w = ops.mx_pack_weight(codes, exps)
    assert w.shape == shape
    c3, e3 = codes.view(-1, *shape[-2:]), exps.view(-1, shape[-2], shape[-1] // 32)
    assert torch.equal(w.codes & 15, c3[..., 0::2]) and torch.equal(w.codes >> 4, c3[..., 1::2])
    for e in range(c3.shape[0]):
        for r in range(shape[-2]):
            for b in range(shape[-1] // 32):
                assert w.scales[e, r // 128, b // 4, r % 32 * 16 + r % 128 // 32 * 4 + b % 4] == e3[e, r, b]


def test_interleave():
    gate, up = torch.arange(2 * 64 * 3).view(2, 64, 3), -torch.arange(2 * 64 * 3).view(2, 64, 3)
    both = ops.mx_interleave(gate, up)
    assert both.shape == (2, 128, 3)
    for i in range(64):
        at = i // 32 * 64 + i % 32
        assert torch.equal(both[:, at], gate[:, i]) and torch.equal(both[:, at + 32], up[:, i])


def test_refusals():
    z = lambda *shape: torch.zeros(shape, dtype=torch.uint8)
    for codes, exps in ((z(4, 48), z(4, 1)), (z(4, 64), z(4, 1)), (z(4, 64).int(), z(4, 2)), (z(64), z(2)), (z(0, 64), z(0, 2)),
                        (z(4, 64), z(3, 2)), (z(2, 4, 64), z(4, 2)), (z(4, 64) + 16, z(4, 2)), (z(4, 64), z(4, 2).int())):
        with pytest.raises(ops.KernelError):
            ops.mx_pack_weight(codes, exps)
    with pytest.raises(ops.KernelError):
        ops.mx_pack_weight(z(96, 64), z(96, 2), glu=True)
    with pytest.raises(ops.KernelError):
        ops.mx_interleave(z(48, 64), z(48, 64))
    with pytest.raises(ops.KernelError):
        ops.mx_interleave(z(64, 64), z(32, 64))
    with pytest.raises(ops.KernelError):
        ops.MxWeight(z(1, 4, 32), z(1, 1, 1, 512), (4, 64))
    w = ops.mx_pack_weight(z(4, 64), z(4, 2))
    for call in (lambda: ops.mx_quantize(torch.zeros(4, 64)), lambda: ops.mx_quantize_weight(torch.zeros(4, 64)),
                 lambda: ops.mx_linear(torch.zeros(4, 64), w)):                     # no CPU path
        with pytest.raises(ops.KernelError):
            call()


def test_forms():
    """Which kernel a product takes, by sizes alone: clusters that share K where a weight has few tiles, single blocks for few rows and experts, pairs of
    blocks for many rows."""
    form = lambda rows, experts, n_out, k, glu=0: ops.lib().hb_mx_gemm_form(rows, experts, n_out, k, glu)
    assert form(1, 1, 5120, 8192) // 1000 in (2, 3) and form(8, 1, 7168, 5120) == 1064 and form(1, 1, 64, 32) == 1064
    assert form(64, 1, 16384, 5120) == 1064 and form(100, 1, 16384, 5120) == 1128 and form(160, 1, 16384, 5120) == 1192
    assert form(256, 1, 5120, 8192) == 1128 and form(512, 1, 5120, 8192) == 1192 and form(256, 1, 16384, 5120) == 1256
    assert form(2048, 1, 16384, 5120) == 0 and form(8192, 1, 5120, 5120) == 0
    assert form(64, 16, 16384, 5120, 1) == 1064 and form(2048, 16, 16384, 5120, 1) == 1128 and form(2100, 16, 5120, 8192) == 1256
    assert form(4096, 16, 5120, 8192) == 1256 and form(12000, 4, 8256, 5152, 1) == 0 and form(12288, 64, 2048, 2048, 1) == 0 and form(12288, 64, 2048, 1024) == 1256
    for rows in (1, 2, 7, 64, 65, 128, 129, 500, 3000, 100000):
        for experts in (1, 2, 64, 1024):
            for n_out in (1, 64, 5120, 200000):
                for k in (32, 256, 288, 8192, 65536):
                    f = form(rows, experts, n_out, k)
                    splits, most = divmod(f, 1000)
                    tiles = (-(-rows // 128) + min(rows, experts) - 1) * -(-n_out // 128)
                    assert f == 0 or (most in (64, 128, 192, 256) and 1 <= splits <= 8 and (splits == 1 or (splits * tiles <= 148 and splits <= -(-k // 256))))
                    assert most != 64 or rows <= 64
    assert form(0, 1, 64, 32) == -1
