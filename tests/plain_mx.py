"""Microscaled 4-bit floats in 64 bits, written from the format: blocks of 32, a power of two each, e2m1 values."""
import torch

STEPS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def two(e):
    """2^e for whole -1022 <= e <= 1023, from its bits (a power function may be off by a rounding)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exponent(x):
    """[..., K] -> e of every block [..., K / 32], from the bits of the largest magnitude; blocks with values that are not finite: 128."""
    top = x.double().abs().unflatten(-1, (-1, 32)).amax(-1)
    bad = ~torch.isfinite(x.double()).unflatten(-1, (-1, 32)).all(-1)
    e = torch.frexp(torch.where(bad, torch.ones_like(top), top))[1].double() - 1 - 2          # 2^(frexp - 1) <= top
    e = torch.where(top > 0, e, torch.full_like(e, -127.0)).clamp(min=-127.0)
    return torch.where(bad, torch.full_like(e, 128.0), e)


def nearest(v):
    """Codes 0 .. 7 of magnitudes in units of 2^e: the nearest step, on a border the even one, the last above it."""
    steps = STEPS.to(v.device)
    distance = (v.unsqueeze(-1) - steps).abs()
    best = distance.amin(-1, keepdim=True)
    near = distance == best
    index = torch.arange(8, device=v.device)
    even = near & (index % 2 == 0)
    return torch.where(near.sum(-1) > 1, even.long().argmax(-1), near.long().argmax(-1))


def quantise(x):
    """[..., K] -> codes uint8 [..., K] and exponents uint8 [..., K / 32]."""
    e = exponent(x)
    unit = two(e.clamp(max=127.0)).unsqueeze(-1)
    y = x.double().unflatten(-1, (-1, 32))
    bad = (e == 128).unsqueeze(-1)
    y = torch.where(bad, torch.zeros_like(y), y)
    codes = nearest((y / unit).abs()) + 8 * (y < 0).long()
    return codes.flatten(-2).to(torch.uint8), (e + 127).to(torch.uint8)


def values(codes, exponents):
    sign = torch.where(codes >= 8, -1.0, 1.0).double()
    unit = two(exponents.to(torch.int64) - 127)
    unit = torch.where(exponents == 255, torch.full_like(unit, float("nan")), unit)
    return sign * STEPS.to(codes.device)[(codes % 8).long()] * unit.repeat_interleave(32, -1)


def held(x):
    return values(*quantise(x))


def unit(gate, up, limit=0.0):
    if limit > 0:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit) + 1.0
        return gate * torch.sigmoid(1.702 * gate) * up
    return gate * torch.sigmoid(gate) * up


def is_quantised(got, act, tol):
    """Whether ``got`` are quantised values of numbers within ``tol`` of ``act`` [..., K]: the block's exponent is one that its largest magnitude,
    give or take ``tol``, has, and every value is the nearest step of one that near, or the last."""
    g, a, t = (v.unflatten(-1, (-1, 32)) for v in (got.double(), act, tol))
    top, slack = a.abs().amax(-1), t.amax(-1)
    fine = torch.zeros(g.shape[:-1], dtype=torch.bool, device=g.device)
    for m in (top - slack, top + slack):
        e = exponent(m.clamp(min=0.0).unsqueeze(-1).expand(*m.shape, 32)).squeeze(-1)
        step = two(e).unsqueeze(-1)
        low, high = ((a + s * t) / step for s in (-1, 1))
        to = lambda v: torch.sign(v) * STEPS.to(v.device)[nearest(v.abs())]
        fine |= ((to(low) * step <= g) & (g <= to(high) * step)).all(-1)
    return fine.all()
