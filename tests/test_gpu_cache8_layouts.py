"""Scales of 8-bit pages in one buffer, keys, values and layers side by side in every order: the calls against those of scales in
buffers of their own."""
from __future__ import annotations

import itertools

import pytest
import torch

from localrouter_amd import cache, ops
from tests.cache8_util import E8, F8
from tests.cache_util import gen, rnd
from tests.test_gpu_cache import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", list(itertools.permutations(range(3))), ids=lambda o: "-".join(("layers", "kv", "pages")[i] for i in o))
def test_scales_side_by_side(order):
    layers, n, ps, HK, g = 3, 6, 32, 2, gen(81)
    kp, vp = (torch.randint(0, 100, (layers, n, ps, HK, 128), generator=g, device="cuda", dtype=torch.uint8).view(F8) for _ in range(2))
    shape = [(layers, 2, n)[i] for i in order]
    one = torch.zeros(*shape, ps // 16, HK, dtype=torch.uint8, device="cuda")
    one = one.permute(*[order.index(i) for i in range(3)], 3, 4)      # [layers, 2, n_pages, groups, heads]
    one.copy_(torch.randint(120, 130, one.shape, generator=g, device="cuda", dtype=torch.uint8))
    side = one.view(E8)
    ks, vs = (one[:, i].clone(memory_format=torch.contiguous_format).view(E8) for i in range(2))
    k2, v2 = kp.view(torch.uint8).clone().view(F8), vp.view(torch.uint8).clone().view(F8)

    def same():
        for x, y in ((kp, k2), (vp, v2), (side[:, 0], ks), (side[:, 1], vs)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    cache.copy_pages_f8(kp, vp, side[:, 0], side[:, 1], ints([0, 3]), ints([4, 5]))
    cache.copy_pages_f8(k2, v2, ks, vs, ints([0, 3]), ints([4, 5]))
    same()
    table, starts, lens = ints([[1, 4], [5, 0]]), ints([0, 20, 23]), ints([50, 30])
    q, k, v = rnd(g, 23, 4, 128), rnd(g, 23, HK, 128), 9 * rnd(g, 23, HK, 128)
    for x in range(layers):
        mine, other = (kp[x], vp[x], side[x, 0], side[x, 1]), (k2[x], v2[x], ks[x], vs[x])
        for p in (mine, other):
            cache.append_f8(None, k, v, *p, table, starts, lens, table_kind=ops.TABLE_NONE)
        assert torch.equal(cache.attention_f8(q, *mine, table, starts, lens), cache.attention_f8(q, *other, table, starts, lens))
    same()
