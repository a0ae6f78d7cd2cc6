"""Every scale byte through attention_f8's kernels: what an element of pages that append_f8 did not write stands for."""
from __future__ import annotations

import pytest
import torch

from localrouter_amd import cache
from tests.cache8_util import E8, F8
from tests.cache_util import gen, rnd
from tests.test_gpu_cache import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [1, 24, 2048])
def test_every_scale_byte(H):
    """A sequence of one key for each byte: its token's result is the key's value. Of few rows a kv head and of many."""
    n = 256
    byte = torch.arange(n, device="cuda", dtype=torch.uint8)
    vp = (torch.arange(n * 16 * 128, device="cuda") % 251).to(torch.uint8).view(n, 16, 1, 128)
    vp[vp & 0x7f == 0x7f] = 1          # (no NaN but the scales')
    kp = torch.zeros_like(vp)
    ks, vs = torch.full((n, 1, 1), 127, dtype=torch.uint8, device="cuda"), byte.view(n, 1, 1).clone()
    q = rnd(gen(1), n, H, 128)
    one, many = ints([1] * n), ints([16] * n)
    args = kp.view(F8), vp.view(F8), ks.view(E8), vs.view(E8), ints([[i] for i in range(n)]), ints(list(range(n + 1)))
    out = cache.attention_f8(q, *args, one, max_rows=1, max_keys=16).double()
    want = vp.view(F8)[:, 0].double() * torch.exp2(byte.double() - 127)[:, None, None]
    size = want.abs()
    normal = (size < 2.0 ** 128) & ((size >= 2.0 ** -126) | (size == 0))
    normal[255] = False
    w, m = want.expand_as(out), normal.expand_as(out)
    assert torch.equal(out[m], w[m])
    assert out[255].isnan().all()
    large = (size >= 2.0 ** 128).expand_as(out)
    large[255] = False
    assert (out[large].sign() == w[large].sign()).all() and out[large].isinf().all()
    small = ((size < 2.0 ** -126) & (size > 0)).expand_as(out)
    # (a value below bf16's normal numbers is rounded to a multiple of 2^-133, or taken for 0: off by less than itself or half of that step,
    # 2^-126 at most either way)
    assert ((out - w).abs()[small] <= 2.0 ** -126).all()
    # a key's scale: scores of 0 times any finite scale, so that the sequence's values have their mean, whatever the byte
    ks[:, 0, 0], vs[:] = byte, 127
    out = cache.attention_f8(q, *args, many, max_rows=1, max_keys=16)
    mean = vp.view(F8).double().mean(1).expand(n, H, 128)
    mag = vp.view(F8).double().abs().mean(1).expand(n, H, 128)
    ok = torch.arange(n) < 255
    assert ((out.double() - mean).abs()[ok] <= (2.0 ** -8 * mean.abs() + 2.0 ** -20 * mag)[ok]).all() and out[255].isnan().all()
