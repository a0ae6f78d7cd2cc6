"""Rows whose sums grow past 2^32, in blocks with padding rows and rows whose sums overflow (attn_packed.hip, attn_cache_wide.hip over pages
of 8 bits): keys of one head many times the queries' size, against 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from localrouter_amd import ops
from tests.cache8_util import exps, scales_of
from tests.cache_util import HALF, gen, ref_rows, rnd
from tests.test_gpu_cache import chain_seen, ints
from tests.test_gpu_cache8 import Batch8
from tests.test_gpu_packed import seen_of, some, sums

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(128.0)


def check_loud(got, q, k, v, seen, what):
    """cache_util's tolerance, with a score's error of 128 products (2^-17 of the sum of |q k|) and of the references that a row went through
    (each off by half an ulp of a number of that size, and there are at most as many as octaves by 32) above and below the fraction bar."""
    ref, mag = ref_rows(q, k, v, seen)
    n, H, D = q.shape
    HK = k.shape[1]
    size = torch.matmul(q.double().abs().cpu().view(n, HK, H // HK, D).permute(1, 2, 0, 3).reshape(HK, -1, D),
                        k.double().abs().cpu().permute(1, 2, 0).contiguous()).amax(-1).view(HK, H // HK, n).permute(2, 0, 1).reshape(n, H, 1)
    err = 2 * (2.0 ** -17 + 2.0 ** -20) * size * SCALE
    tol = HALF * ref.abs() + (2 * HALF + 2.0 ** -11 + err) * mag + 1e-30
    d = (got.double().cpu() - ref).abs()
    assert (d <= tol).all(), f"{what}: {int((d > tol).sum())} values off, worst {float((d / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("times", [8, 24, 64])
@pytest.mark.parametrize("lens,H,HK", [([637, 129, 33, 1, 700], 32, 8), ([333] * 9, 16, 16), ([2001, 70], 24, 8)], ids=["r4", "r1", "r3"])
def test_packed(lens, H, HK, times):
    g, T = gen(101), sum(lens)
    q, k, v = rnd(g, T, H, 128), rnd(g, T, HK, 128), rnd(g, T, HK, 128)
    k[:, 0] *= times
    out = ops.attention_packed(q, k, v, ints(sums(lens)))
    st = sums(lens)
    for b, n in enumerate(lens):
        at = some(n, 3)
        rows, s = [st[b] + i for i in at], slice(st[b], st[b] + n)
        check_loud(out[rows], q[rows], k[s], v[s], seen_of(n)[at], f"sequence {b}")


@pytest.mark.parametrize("times", [3, 5, 6])
@pytest.mark.parametrize("news,lens,H,HK", [([705], [5700], 32, 8), ([333, 250], [3000, 2500], 56, 8), ([701, 130], [1500, 130], 48, 2)],
                         ids=["r4", "r7", "r24"])
def test_chunks(news, lens, H, HK, times):
    B = Batch8(102, news, lens, 32, HK)
    e = exps(B.ks)
    e[:, :, 0] += times
    B.ks = scales_of(e)
    q = rnd(B.g, sum(news), H, 128)
    out = B.attend(q, max_rows=max(news), max_keys=max(lens))
    for b, n in enumerate(news):
        at = some(n, 3)
        rows = [B.st[b] + i for i in at]
        k, v = B.rows(b)
        check_loud(out[rows], q[rows], k, v, chain_seen(n, lens[b])[at], f"sequence {b}")
