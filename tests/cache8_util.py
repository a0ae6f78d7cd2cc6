"""Shared by the tests of the cache in 8-bit pages: the format restated with torch's own conversions, and a plain append."""
from __future__ import annotations

import torch

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
GROUP = 16


def exponent(a):
    """The least e with a <= 448 * 2^e, in [-100, 119], for fp64 a >= 0."""
    m, x = torch.frexp(a)
    return torch.where(a > 0, torch.where(m > 0.875, x - 8, x - 9), -100).clamp(-100, 119)


def to_f8(x):
    """fp64 -> e4m3 to nearest even, one rounding (what goes through fp32 on the way here is exact there); not finite -> NaN."""
    bad = ~torch.isfinite(x)
    x = x.clamp(-448, 448)
    step = torch.exp2((torch.frexp(x.abs())[1] - 1).clamp(min=-6).double() - 3)
    y = (torch.round(x / step) * step).float()
    return torch.where(bad, float("nan"), y).to(F8)


def pack(x):
    """A pool [..., page_size, HK, 128] -> its 8-bit pages and scales, each group of 16 rows at the least scale that holds it."""
    y = x.double().unflatten(-3, (-1, GROUP))
    e = exponent(torch.where(torch.isfinite(y), y.abs(), 0.0).amax((-3, -1)))            # [..., groups, HK]
    q = to_f8(y * torch.exp2(-e.double())[..., None, :, None]).flatten(-4, -3)
    return q, (e + 127).to(torch.uint8).view(E8)


def scales_of(e):
    return (e + 127).to(torch.uint8).view(E8)


def exps(scales):
    return scales.view(torch.uint8).int() - 127


def values(pages, scales):
    """What 8-bit pages stand for, in fp64: e4m3 values times powers of two."""
    return pages.float().double() * torch.exp2(exps(scales).double()).repeat_interleave(GROUP, -2)[..., None]
