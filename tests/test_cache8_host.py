"""The cache in 8-bit pages on the CPU: the bindings agree with the header, bad arguments are refused before any GPU call, and the
restatement of the format that the GPU tests compare with agrees with torch's conversions. No compute calls."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

from localrouter_amd import cache
from tests.cache8_util import F8, exponent, pack, to_f8, values
from tests.test_zig_bindings import C_KIND, ZIG_KIND

ROOT = Path(__file__).resolve().parent.parent
BAD = 1   # hipErrorInvalidValue
# fake, well-aligned device addresses, far apart from each other
Q, K, V, O, KP, VP, WS, KS, VS = (x << 32 for x in (1, 2, 3, 4, 5, 6, 7, 20, 21))
I1, I2, I3, I4, I5, I6 = (x << 32 for x in (8, 9, 10, 11, 12, 13))


def test_bindings_match_the_header():
    text = re.sub(r"/\*.*?\*/", "", cache.HEADER_F8.read_text(), flags=re.S)
    head = {}
    for m in re.finditer(r"\b(int|size_t)\s+(lr_\w+)\s*\(([^)]*)\)\s*;", text):
        args = [a.strip() for a in m.group(3).split(",")]
        head[m.group(2)] = (C_KIND[m.group(1)], ["ptr" if "*" in a or a.startswith("lr_stream_t") else
                                                 C_KIND[a.rsplit(" ", 1)[0].replace("const ", "")] for a in args])
    kinds = {cache._P: "ptr", cache._I: "i32", cache._I64: "i64", cache._F: "f32", cache._SZ: "usize"}
    assert len(head) == 4
    assert {n: (kinds[r], [kinds[a] for a in args]) for n, (r, args) in cache.SIGNATURES_F8.items()} == head
    assert all(hasattr(cache.lib(), n) for n in head)
    zig = {}
    for m in re.finditer(r'pub extern "lr_attn" fn (lr_\w+)\((.*?)\)\s*(\w+);', (ROOT / "src/engines/hip/lr_cache8.zig").read_text(),
                         flags=re.S):
        zig[m.group(1)] = (ZIG_KIND[m.group(3)], [ZIG_KIND[a.split(":", 1)[1].strip()]
                                                  for a in m.group(2).replace("\n", " ").split(",")])
    assert zig == head


# page 16 rows of 2 heads; a page's scales: 2 bytes
POOL = dict(page_stride=4096, row_stride=256, head_stride=128, n_pages=100, page_size=16)
POOL_BAD = [dict(n_pages=0), dict(page_size=8), dict(page_size=24), dict(page_size=0), dict(page_stride=2048), dict(page_stride=4104),
            dict(row_stride=128), dict(row_stride=264), dict(head_stride=64), dict(head_stride=136), dict(row_stride=1 << 23, page_stride=1 << 28),
            dict(n_pages=1 << 30, page_stride=1 << 40)]
SCALES_BAD = [dict(ks=0), dict(vs=0), dict(sps=1), dict(sps=-4), dict(sps=1 << 47), dict(vs=KS), dict(vs=KS + 1, sps=4),
              dict(ks=KP + 100), dict(vs=VP + 4096 * 99 + 4000)]


def _append(**kw):
    a = dict(q=Q, k=K, v=V, qrs=1024, krs=256, vrs=256, qo=O, qors=1024, k_pages=KP, v_pages=VP, **POOL, ks=KS, vs=VS, sps=2, table=I1,
             table_stride=50, table_pages=50, starts=I2, lens=I3, pos=None, B=3, T=70, H=8, HK=2, qw=None, kw=None, kind=1, ta=I4, tb=I5,
             trs=64, trows=100, pairing=0, rot=128, eps=1e-6, stream=None)
    a.update(kw)
    return cache.lib().lr_cache_append_f8(*a.values())


@pytest.mark.parametrize("kw", POOL_BAD + SCALES_BAD + [
    dict(q=Q + 8), dict(qo=0), dict(k=0), dict(v=0), dict(krs=128), dict(vrs=260), dict(qors=512), dict(T=0), dict(H=0), dict(HK=0),
    dict(eps=-1.0), dict(eps=float("inf")), dict(k_pages=KP + 8), dict(v_pages=KP), dict(v_pages=KP + 128), dict(table=0),
    dict(table_stride=49), dict(table_pages=0), dict(table_pages=1 << 27, table_stride=1 << 27), dict(starts=0), dict(lens=0),
    dict(lens=I3 + 2), dict(pos=I6 + 1), dict(B=0), dict(B=65536), dict(qw=I6 + 4), dict(kw=I6 + 8), dict(kind=7), dict(ta=0),
    dict(tb=0), dict(trs=32), dict(trows=0), dict(pairing=2), dict(rot=130), dict(pairing=1, rot=24), dict(qo=Q + 256), dict(qo=K),
    dict(k=KP), dict(q=VP), dict(qo=VP), dict(ks=K), dict(vs=V + 10), dict(ks=Q), dict(vs=O), dict(T=1 << 30, HK=2, H=64, qrs=8192, qors=8192),
], ids=str)
def test_append_refuses(kw):
    assert _append(**kw) == BAD


def _attend(**kw):
    a = dict(q=Q, qrs=1024, out=O, ors=1024, k_pages=KP, v_pages=VP, **POOL, ks=KS, vs=VS, sps=2, table=I1, table_stride=50,
             table_pages=50, starts=I2, lens=I3, B=3, T=70, max_rows=40, max_keys=800, H=8, HK=2, tree=None, words=0, window=0, sinks=0,
             scale=0.088, ws=WS, wsb=1 << 31, stream=None)
    a.update(kw)
    return cache.lib().lr_cache_attention_f8(*a.values())


ONE = dict(T=3, max_rows=1, max_keys=100000)   # split over the keys


@pytest.mark.parametrize("kw", POOL_BAD + SCALES_BAD + [
    dict(q=0), dict(out=0), dict(qrs=1023), dict(ors=1000), dict(H=9), dict(HK=0), dict(B=0), dict(B=65536), dict(T=0), dict(max_rows=0),
    dict(max_keys=0), dict(max_keys=(1 << 30) + 1), dict(max_rows=1 << 30), dict(max_rows=1 << 28), dict(window=-1), dict(sinks=-1),
    dict(scale=0.0), dict(scale=float("nan")), dict(tree=I4, words=0), dict(tree=I4, words=65), dict(tree=I4 + 4, words=1), dict(out=Q),
    dict(out=KP), dict(out=VP + 512), dict(out=KS), dict(out=VS), dict(table=0), dict(starts=I2 + 1), dict(lens=0), dict(table_stride=1),
    dict(ws=0, **ONE), dict(wsb=8, **ONE), dict(ws=WS + 16, **ONE), dict(ws=KP, **ONE), dict(ws=O, **ONE), dict(ws=KS, **ONE),
], ids=str)
def test_attention_refuses(kw):
    assert _attend(**kw) == BAD


def test_workspace_sizes():
    assert cache.attention_f8_ws_bytes(1, 1, 1, 100000, 8, 8, 8) == 0      # (pages of 8 rows: refused)
    need = cache.attention_f8_ws_bytes(1, 1, 1, 100000, 8, 2, 16)
    assert need > 0 and need % 256 == 0
    assert cache.attention_f8_ws_bytes(1, 1, 1, 20, 8, 2, 16) == 0
    with pytest.raises(ValueError):
        cache.attention_f8_ws_bytes(1, 1, 1, 1 << 40, 8, 2, 16)


def _copy(**kw):
    a = dict(k_pages=KP, v_pages=VP, layers=3, layer_stride=1 << 20, **POOL, HK=2, ks=KS, vs=VS, sls=200, sps=2, src=I1, dst=I2, n=5,
             stream=None)
    a.update(kw)
    return cache.lib().lr_cache_copy_pages_f8(*a.values())


@pytest.mark.parametrize("kw", POOL_BAD + SCALES_BAD + [
    dict(layers=0), dict(layer_stride=64), dict(layer_stride=1 << 12), dict(HK=0), dict(sls=100), dict(sls=1), dict(sps=6, sls=1),
    dict(sps=6, sls=3), dict(src=0), dict(dst=I2 + 1), dict(n=0), dict(vs=KS + 2), dict(ks=KP + (3 << 20) - (1 << 20)),
], ids=str)
def test_copy_refuses(kw):
    assert _copy(**kw) == BAD


def test_tensors_on_the_host_are_refused():
    kp, vp = (torch.zeros(4, 16, 2, 128).to(F8) for _ in range(2))
    ks, vs = (torch.zeros(4, 1, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2))
    x, i = torch.zeros(3, 2, 128, dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        cache.append_f8(None, x, x, kp, vp, ks, vs, i[None], i, i, table_kind=0)
    with pytest.raises(ValueError, match="GPU"):
        cache.attention_f8(x, kp, vp, ks, vs, i[None], i, i)
    with pytest.raises(ValueError, match="GPU"):
        cache.copy_pages_f8(kp, vp, ks, vs, i, i)


def test_the_format_restated():
    """The exponent is the least that holds its value, at and beside the borders; one rounding to nearest even agrees with torch's."""
    a = torch.tensor([448.0 * 2.0 ** e for e in range(-120, 121, 7)], dtype=torch.float64)
    for x, up in ((a, 0), (a * (1 + 2.0 ** -30), 1), (a * (1 - 2.0 ** -30), 0)):
        want = torch.arange(-120, 121, 7) + up
        assert torch.equal(exponent(x), want.clamp(-100, 119).to(exponent(x).dtype))
    assert exponent(torch.zeros(1, dtype=torch.float64)).item() == -100
    g = torch.Generator().manual_seed(3)
    x = torch.cat([torch.randn(40000, generator=g) * s for s in (0.004, 0.1, 3.0, 150.0)]).clamp(-448, 448)
    x = torch.cat([x, torch.arange(-448, 449).float(), torch.arange(-64, 65).float() / 1024])
    assert torch.equal(to_f8(x.double()).view(torch.uint8), x.to(F8).view(torch.uint8))
    assert to_f8(torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=torch.float64)).float().isnan().all()
    y = torch.randn(3, 32, 2, 128, generator=g).to(torch.bfloat16) * torch.exp2(torch.randint(-30, 30, (3, 32, 2, 1), generator=g))
    q, s = pack(y)
    d, top = (values(q, s) - y.double()).abs(), y.double().abs().unflatten(1, (-1, 16)).amax((2, 4)).repeat_interleave(16, 1)[..., None]
    assert (d <= 2.0 ** -4 * y.double().abs() + top * 2.0 ** -17).all()   # half a step, or half of the smallest (2^-10 of 224 and more)
