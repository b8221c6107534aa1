"""What of the 4-bit weights and the 4-bit cache runs without a GPU: the layout, the quantisation, the sizes, the refusals."""
import pytest
import torch

from hi_b200.kernels import ops
from plain_four_bit import unpack_weight, weight_values


@pytest.mark.parametrize("m,k,group", [(1, 32, 32), (16, 128, 128), (17, 192, 64), (40, 416, 32), (33, 320, 64), (5, 384, 128)])
def test_packed_weights_hold_their_codes(m, k, group):
    g = torch.Generator().manual_seed(m * k)
    codes = torch.randint(0, 16, (m, k), generator=g).to(torch.uint8)
    scales = torch.rand(m, k // group, generator=g).to(torch.bfloat16)
    w = ops.pack_weight(codes, scales)
    assert w.shape == (m, k) and w.group == group and w.blocks.shape == (-(-m // 16), -(-k // 128), 1024 + 32 * (128 // group))
    got_codes, got_scales = unpack_weight(w)
    assert torch.equal(got_codes, codes) and torch.equal(got_scales, scales)
    # what lies behind the matrix counts as nothing
    if k % 128:
        assert w.blocks[:, -1, :1024].view(-1, 16, 4, 4, 4)[:, :, :, -1].eq(0x88).all()


@pytest.mark.parametrize("group", ops.FOUR_BIT_GROUPS)
def test_quantised_weights_are_within_half_a_step(group):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(19, 384, generator=g) * torch.exp(torch.randn(19, 1, generator=g))
    w[3, :group] = 0.0
    codes, scales = unpack_weight(ops.quantize_weight(w, group))
    step = scales.double().repeat_interleave(group, 1)
    # half a step, and seven steps of a scale that was rounded by up to 2^-8 (the largest weight lies there)
    assert ((weight_values(codes, scales) - w.double()).abs() <= step * (0.5 + 7 * 2.0 ** -8)).all()
    assert (codes[3, :group] == 8).all() and (scales[3, 0] == 0)
    bf16 = unpack_weight(ops.quantize_weight(w.to(torch.bfloat16), group))
    assert torch.equal(bf16[0], unpack_weight(ops.quantize_weight(w.to(torch.bfloat16).float(), group))[0])
    w[2, 5], w[4, -1] = float("inf"), float("nan")
    values = weight_values(*unpack_weight(ops.quantize_weight(w, group)))
    assert values[2, :group].isnan().all() and values[4, -group:].isnan().all() and int(values.isnan().sum()) == 2 * group


def test_refusals_without_a_gpu():
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 2, dtype=torch.bfloat16)
    for c, s in ((codes.int(), scales), (codes, scales.float()), (codes, scales[:3]), (codes, scales[:, :0]),
                 (codes[:, :48], scales), (codes[:0], scales[:0]), (codes, torch.ones(4, 4, dtype=torch.bfloat16)), (codes[0], scales[0])):
        with pytest.raises(ops.KernelError):
            ops.pack_weight(c, s)
    for w, group in ((torch.ones(4, 48), 32), (torch.ones(4, 64), 16), (torch.ones(64), 64), (torch.ones(4, 64, dtype=torch.int32), 64)):
        with pytest.raises(ops.KernelError):
            ops.quantize_weight(w, group)
    w = ops.pack_weight(codes, scales)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.four_bit_linear(torch.ones(2, 64, dtype=torch.bfloat16), w)
    for page, hd in ((64, 96), (48, 128), (8, 64), (0, 64), (-64, 64)):
        with pytest.raises(ops.KernelError):
            ops.four_bit_page_bytes(page, hd)
    assert ops.four_bit_page_bytes(64, 128) == 64 * 160 and ops.four_bit_page_bytes(16, 64) == 16 * 80
    pages = torch.zeros(2, 2, 64 * 160, dtype=torch.uint8)
    i32 = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.decode_attention_4bit(torch.zeros(1, 4, 128, dtype=torch.bfloat16), pages, i32, i32[0], i32[0], 0, 0, 1.0, 1)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.expand_pages_4bit(pages, 128, i32, i32[0], i32[0], [0], [1])
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.qkv_post_4bit(torch.zeros(1, 8 * 128, dtype=torch.bfloat16), 4, 2, 128, i32[0], None, False, False, 1e-6, None, i32[0], i32, pages)


def test_cuts_cover_the_keys():
    for tiles in (1, 2, 3, 7, 16, 63, 100, 513, 2048, 40000):
        for groups, hd in ((1, 64), (8, 128), (40, 64), (64, 128), (512, 64), (8192, 128)):
            size, splits = ops._four_bit_splits(tiles, groups, hd)
            assert size >= 1 and splits >= 1 and size * splits >= tiles and size * (splits - 1) < tiles


@pytest.mark.parametrize("shape,group,blocks", [
    ((17, 100), 64, (2, 1, 1088)), ((16, 128), 64, (2, 1, 1088)), ((16, 128), 64, (1, 1, 1056)), ((16, 256), 128, (1, 1, 1056)),
    ((16, 128), 16, (1, 1, 1280)), ((0, 128), 128, (0, 1, 1056)), ((33, 64), 32, (2, 1, 1152))])
def test_blocks_that_are_not_the_weights(shape, group, blocks):
    with pytest.raises(ops.KernelError):
        ops.FourBitWeight(torch.zeros(blocks, dtype=torch.uint8), shape, group)


def test_blocks_that_are():
    w = ops.FourBitWeight(torch.zeros(3, 1, 1152, dtype=torch.uint8), (33, 64), 32)
    assert w.shape == (33, 64) and w.group == 32
    for blocks in (w.blocks.to(torch.int8), torch.zeros(3, 2, 1152, dtype=torch.uint8)[:, :1]):
        with pytest.raises(ops.KernelError):
            ops.FourBitWeight(blocks, (33, 64), 32)
