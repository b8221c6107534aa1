"""Plain forms of the 4-bit weight and of the 4-bit cache, in torch, on any device."""
import math

import torch

GROUP = 32


def unpack_weight(weight):
    """Codes uint8 [M, K] and scales bfloat16 [M, K / group] out of a FourBitWeight's bytes, bit by bit."""
    m, k = weight.shape
    blocks, per = weight.blocks, 128 // weight.group
    tiles, chunks, _ = blocks.shape
    words = blocks[..., :1024].reshape(tiles, chunks, 16, 4, 4, 4).to(torch.int64)      # [.., row, lane, word, byte]
    words = sum(words[..., b] << (8 * b) for b in range(4))
    codes = torch.zeros(tiles * 16, chunks * 128, dtype=torch.uint8, device=blocks.device)
    view = codes.view(tiles, 16, chunks, 4, 4, 8)                                       # [.., word, lane, eight k]
    for e in range(8):
        at = e // 2 if e % 2 == 0 else 4 + e // 2
        view[..., e] = ((words >> (4 * at)) & 15).to(torch.uint8).permute(0, 2, 1, 4, 3)
    scales = blocks[..., 1024:].contiguous().view(torch.bfloat16).reshape(tiles, chunks, 16, per)
    scales = scales.transpose(1, 2).reshape(tiles * 16, chunks * per)
    return codes[:m, :k], scales[:m, : k // weight.group]


def weight_values(codes, scales, dtype=torch.float64):
    group = codes.shape[1] // scales.shape[1]
    return (codes.to(dtype) - 8) * scales.to(dtype).repeat_interleave(group, dim=1)


def quantise(x):
    """[..., dim] -> codes uint8 [..., dim], scale and low bfloat16 [..., dim / 32], of the values in bfloat16."""
    y = x.to(torch.bfloat16).to(torch.float32).unflatten(-1, (-1, GROUP))
    whole = torch.isfinite(y).all(-1)
    low = y.amin(-1)
    scale = ((y.amax(-1) - low) / 15.0).to(torch.bfloat16)
    step = scale.to(torch.float32).unsqueeze(-1)
    codes = torch.where(step > 0, ((y - low.unsqueeze(-1)) / step).round().clamp(0, 15), torch.zeros_like(y))
    codes = torch.where(whole.unsqueeze(-1), codes, torch.zeros_like(codes))
    nan = torch.full_like(scale, float("nan"))
    return codes.to(torch.uint8).flatten(-2), torch.where(whole, scale, nan), torch.where(whole, low.to(torch.bfloat16), nan)


def values(parts, dtype=torch.float64):
    codes, scale, low = parts
    y = codes.to(dtype).unflatten(-1, (-1, GROUP))
    return (scale.to(dtype).unsqueeze(-1) * y + low.to(dtype).unsqueeze(-1)).flatten(-2)


def visible(pos, keys, chunk=0, window=0, keep=0):
    """[tokens, keys] which keys a token at each position reads."""
    at = torch.arange(keys, device=pos.device)
    p = pos.long().unsqueeze(1)
    low = torch.zeros_like(p)
    if chunk:
        low = p // chunk * chunk
    if window:
        low = (p - window + 1).clamp(min=0)
    return (at <= p) & ((at >= low) | (at < keep))


def attention(q, k, v, seen, scale, sink=None):
    """float64: q [n, heads, dim], k and v [keys, kv heads, dim], seen [n, keys]; ``sink``: the scores of the extra term [heads].
    Returns the result and what it would be with every |p v| instead of p v (what roundings of the weights are relative to)."""
    per = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(per, 1), v.repeat_interleave(per, 1)
    s = torch.einsum("nhd,thd->nht", q.double(), k.double()) * scale
    s = s.masked_fill(~seen.unsqueeze(1), -math.inf)
    top = s.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink.double().view(1, -1, 1))
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink.double().view(1, -1, 1) - top)
    p = p / total
    return torch.einsum("nht,thd->nhd", p, v.double()), torch.einsum("nht,thd->nhd", p, v.double().abs())
