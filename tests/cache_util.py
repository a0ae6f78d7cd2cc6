"""Shared by the tests of the paged cache and the windowed attention: a 64-bit attention over exactly the keys a token sees,
and the tolerance that the arithmetic allows."""
from __future__ import annotations

import math

import torch

# Per element, with A = sum_j p_j |v_j| / sum_j p_j: the output's rounding to bf16 (half a step: 2^-8 relative), the rounding
# of P to bf16 (2^-8 of each p_j in the sum of products, and through the row sum of the rounded P once more), and 2^-10 A for
# fp32: a score's 128 products of |q k| below 2^8 in all are off by at most 128 * 2^-24 * 2^8 * scale < 2^-12 relative in p_j,
# above and below the fraction bar, and sums of at most 2^13 terms by 2^-11.
HALF = 2.0 ** -8


def ref_rows(q, k, v, seen, scale=1.0 / math.sqrt(128.0)):
    """q [n, H, D], k / v [m, HK, D], seen [n, m] bool -> (out, A), both fp64 [n, H, D] on the CPU. Keys that a token does not
    see are not touched; a token that sees none gets zeros."""
    q, k, v, seen = q.double().cpu(), k.double().cpu(), v.double().cpu(), seen.cpu()
    n, H, D = q.shape
    HK = k.shape[1]
    out, mag = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    for i in range(n):
        at = seen[i].nonzero()[:, 0]
        if not len(at):
            continue
        ks = k[at].permute(1, 2, 0).contiguous()                    # [HK, D, m]
        vs = v[at].permute(1, 0, 2).contiguous()                    # [HK, m, D]
        s = torch.matmul(q[i].view(HK, H // HK, D), ks) * scale
        p = torch.softmax(s, -1)
        out[i] = torch.matmul(p, vs).reshape(H, D)
        mag[i] = torch.matmul(p, vs.abs()).reshape(H, D)
    return out, mag


def check_rows(got, ref, mag, what=""):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    inf = ref.isinf()
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities differ"
    fine = torch.isfinite(ref)
    tol = HALF * ref.abs() + (2 * HALF + 2.0 ** -10) * mag + 1e-30
    d = (got - ref).abs()
    over = (d > tol) & fine
    assert not over.any(), f"{what}: {int(over.sum())} values off, worst {float((d / tol)[fine].max()):.2f} of the tolerance"


def window_seen(w, nkeys, p0, window, sinks, frame):
    f = (p0 + torch.arange(w))[:, None] // frame
    j = torch.arange(nkeys)[None]
    return (j // frame <= f) & ((j // frame > f - window) | (j < sinks))


def rnd(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g
