"""The queries of append_f8, a pass of their own beside the 8-bit rows: against the bf16 append's, bit for bit, and against 64 bits."""
from __future__ import annotations

import pytest
import torch

from localrouter_amd import cache, ops
from tests.test_gpu_cache import ints, rnd
from tests.test_gpu_cache8 import BF16, Batch8, angles, turned

pytestmark = pytest.mark.gpu

NONE, CS, M32, M16 = ops.TABLE_NONE, ops.TABLE_COSSIN_F32, ops.TABLE_MAT2_F32, ops.TABLE_MAT2_BF16


@pytest.mark.parametrize("kind,pairing,rot", [(NONE, 0, 128), (CS, 0, 128), (CS, 1, 128), (CS, 1, 32), (CS, 0, 50), (M32, 1, 96), (M32, 0, 128),
                                              (M16, 0, 128), (M16, 1, 64)])
@pytest.mark.parametrize("news,lens,lead", [([21, 3], [50, 3], 0), ([2, 0, 1] * 30, [9, 4, 17] * 30, 0), ([1] * 65, list(range(1, 66)), 3),
                                            ([3] * 64, [40] * 64, 1)], ids=["2seq", "90seq", "65seq", "64seq"])
@pytest.mark.parametrize("given", [False, True])
def test_queries(kind, pairing, rot, news, lens, lead, given):
    """Table rows from `positions` or the lengths, batches whose search is the lanes' own (at most 64 sequences) and larger ones; rows of no
    sequence, tokens whose row is not one of the table's and those whose page the pool does not have stay as they were."""
    H, HK, n = 5, 2, 60
    B = Batch8(32, news, lens, 16, HK)
    T = lead + sum(news)
    q, k, v = rnd(B.g, T, H, 128), rnd(B.g, T, HK, 128), rnd(B.g, T, HK, 128)
    w = torch.rand(128, generator=B.g, device="cuda") + 0.5
    starts = B.starts + lead
    slot = torch.cat([torch.arange(L - m, L) for m, L in zip(news, lens)]).cuda()
    pos = torch.randint(-1, n + 1, (T,), generator=B.g, device="cuda") if given else torch.cat([torch.zeros(lead, device="cuda").long(), slot])
    table_b = [list(r) for r in B.table]
    table_b[0][0] = B.n_pages
    t = ints(table_b)
    live = torch.ones(T, dtype=torch.bool, device="cuda")
    live[:lead] = False
    if kind != NONE:
        live &= (pos >= 0) & (pos < n)
    first = torch.arange(lead, lead + news[0], device="cuda")
    live[first[slot[:news[0]] < 16]] = False
    c, s = angles(n)
    tab = (c, s)
    if kind in (M32, M16):
        m = torch.stack([c, -s, s, c], -1)[:, :rot // 2].flatten(1)
        if kind == M16:
            m = m.to(BF16)
            c, s = m.view(n, -1, 4)[..., 3].float(), m.view(n, -1, 4)[..., 2].float()
        tab = (m.contiguous(), None)
    kw = dict(q_norm=w, table_kind=kind, table=None if kind == NONE else tab, positions=pos.int() if given else None, pairing=pairing, rot=rot)
    out, other = (torch.full((T, H, 128), 7.0, dtype=BF16, device="cuda") for _ in range(2))
    cache.append_f8(q, k, v, B.kp, B.vp, B.ks, B.vs, t, starts, B.lens, out, **kw)
    kp, vp = (torch.zeros(B.n_pages, 16, HK, 128, dtype=BF16, device="cuda") for _ in range(2))
    cache.append(q, k, v, kp, vp, t, starts, B.lens, other, **kw)
    assert live.any() and (out[~live] == 7.0).all() and torch.equal(out, other)
    y, off = turned(q, w, None if kind == NONE else (c, s), pos.clamp(0, n - 1), pairing, rot)
    d = (out.double() - y).abs()[live]
    assert (d <= (off + 2.0 ** -8 * (y.abs() + off))[live]).all()   # (fp32's errors, and half a step of bf16)
    mine = q.clone()
    cache.append_f8(mine, k, v, B.kp, B.vp, B.ks, B.vs, t, starts, B.lens, mine, **kw)
    assert torch.equal(mine, torch.where(live[:, None, None], out, q))
