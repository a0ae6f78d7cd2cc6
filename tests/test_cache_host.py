"""The paged cache and the windowed attention on the CPU: the ctypes and Zig bindings agree with the headers, bad arguments are
refused before any GPU call, and the page bookkeeping. No compute calls."""
from __future__ import annotations

import random
import re
from pathlib import Path

import pytest
import torch

from localrouter_amd import _lib, cache, ops
from tests.test_zig_bindings import C_KIND, ZIG_KIND

ROOT = Path(__file__).resolve().parent.parent
BAD = 1   # hipErrorInvalidValue
# fake, well-aligned device addresses, far apart from each other
Q, K, V, O, KP, VP, WS = (x << 32 for x in (1, 2, 3, 4, 5, 6, 7))
I1, I2, I3, I4, I5, I6 = (x << 32 for x in (8, 9, 10, 11, 12, 13))


def _header_kinds():
    text = re.sub(r"/\*.*?\*/", "", cache.HEADER.read_text(), flags=re.S)
    out = {}
    for m in re.finditer(r"\b(int|size_t)\s+(lr_\w+)\s*\(([^)]*)\)\s*;", text):
        args = [a.strip() for a in m.group(3).split(",")]
        out[m.group(2)] = (C_KIND[m.group(1)], ["ptr" if "*" in a or a.startswith("lr_stream_t") else
                                                C_KIND[a.rsplit(" ", 1)[0].replace("const ", "")] for a in args])
    return out


def test_bindings_match_the_header():
    kinds = {cache._P: "ptr", cache._I: "i32", cache._I64: "i64", cache._F: "f32", cache._SZ: "usize"}
    head = _header_kinds()
    assert len(head) == 5
    assert {n: (kinds[r], [kinds[a] for a in args]) for n, (r, args) in cache.SIGNATURES.items()} == head
    assert all(hasattr(cache.lib(), n) for n in head)
    zig = {}
    text = (ROOT / "src/engines/hip/lr_cache.zig").read_text()
    for m in re.finditer(r'pub extern "lr_attn" fn (lr_\w+)\((.*?)\)\s*(\w+);', text, flags=re.S):
        zig[m.group(1)] = (ZIG_KIND[m.group(3)], [ZIG_KIND[a.split(":", 1)[1].strip()]
                                                  for a in m.group(2).replace("\n", " ").split(",")])
    assert zig == head


def _window(**kw):
    a = dict(q=Q, k=K, v=V, out=O, p0=0, W=300, H=8, HK=2, nkeys=700, window=64, sinks=4, frame=1, scale=0.088, qrs=1024,
             krs=256, vrs=256, ors=1024, ws=WS, wsb=1 << 31, stream=None)
    a.update(kw)
    return _lib.load().lr_attention_window_bf16(*a.values())


@pytest.mark.parametrize("kw", [
    dict(q=0), dict(v=0), dict(out=0), dict(W=0), dict(H=9), dict(HK=0), dict(nkeys=0), dict(window=0), dict(window=-3),
    dict(sinks=-1), dict(frame=0), dict(scale=0.0), dict(scale=float("nan")), dict(p0=-1), dict(p0=(1 << 30) - 100),
    dict(nkeys=(1 << 30) + 1), dict(q=Q + 8), dict(qrs=1023), dict(krs=128), dict(vrs=252), dict(ors=1020),
    dict(out=Q), dict(out=K + 4096), dict(out=V + 256), dict(W=1, H=2, nkeys=100000, window=100000, ws=0),
    dict(W=1, H=2, nkeys=100000, window=100000, wsb=8), dict(W=1, H=2, nkeys=100000, window=100000, ws=WS + 16),
    dict(W=1, H=2, nkeys=100000, window=100000, ws=K),
], ids=str)
def test_window_refuses(kw):
    assert _window(**kw) == BAD


def test_window_workspace_sizes():
    L = _lib.load()
    assert L.lr_attention_window_ws_bytes(0, 8, 2, 700, 64, 4, 1) == 0
    assert ops.attention_window_ws_bytes(16384, 32, 32, 16384, window=4, sinks=1024, frame=1024) == 0   # fills the GPU
    # one token over many keys is split: fp32 rows of 128 and (reference, sum) a range
    need = ops.attention_window_ws_bytes(1, 8, 2, 100000, window=100000)
    assert need > 0 and need % 256 == 0
    # a window bounds what is split, whatever lies before it
    assert ops.attention_window_ws_bytes(1, 8, 2, 1 << 29, window=64) <= ops.attention_window_ws_bytes(1, 8, 2, 512, window=512)


@pytest.mark.parametrize("name", ["w", "heads", "kv_heads", "nkeys", "window", "sinks", "frame"])
@pytest.mark.parametrize("far", [1 << 32, -(1 << 33), 1 << 31])
def test_window_workspace_of_numbers_past_32_bits(name, far):
    """Refused by name, not cut to some other call's workspace."""
    kw = dict(w=1, heads=8, kv_heads=2, nkeys=100000, window=100000, sinks=0, frame=1)
    assert ops.attention_window_ws_bytes(**kw) > 0
    with pytest.raises(ValueError, match=f"^{name}: a 32-bit number"):
        ops.attention_window_ws_bytes(**dict(kw, **{name: kw[name] + far}))


@pytest.mark.parametrize("name", ["B", "T", "max_rows", "max_keys", "heads", "kv_heads", "page_size", "window", "sinks"])
@pytest.mark.parametrize("far", [1 << 32, -(1 << 33), 1 << 31])
def test_cache_workspace_of_numbers_past_32_bits(name, far):
    kw = dict(B=1, T=1, max_rows=1, max_keys=30000, heads=8, kv_heads=2, page_size=16, window=0, sinks=0)
    assert cache.attention_ws_bytes(**kw) > 0
    with pytest.raises(ValueError, match=f"^{name}: a 32-bit number"):
        cache.attention_ws_bytes(**dict(kw, **{name: kw[name] + far}))


def _attend(**kw):
    a = dict(q=Q, qrs=1024, out=O, ors=1024, kp=KP, vp=VP, ps=4096, rs=256, hs=128, n_pages=40, page=16, table=I1, trs=10,
             tp=10, starts=I2, lens=I3, B=3, T=12, rows=6, keys=160, H=8, HK=2, tree=0, words=0, window=0, sinks=0,
             scale=0.088, ws=WS, wsb=1 << 30, stream=None)
    a.update(kw)
    return cache.lib().lr_cache_attention_bf16(*a.values())


@pytest.mark.parametrize("kw", [
    dict(q=0), dict(out=0), dict(kp=0), dict(vp=0), dict(table=0), dict(starts=0), dict(lens=0), dict(B=0), dict(B=70000),
    dict(T=0), dict(rows=0), dict(keys=0), dict(H=7), dict(HK=0), dict(page=12), dict(page=0), dict(page=1 << 17),
    dict(n_pages=0), dict(kp=KP + 8), dict(ps=4090), dict(rs=120), dict(hs=64), dict(hs=124), dict(rs=128),
    dict(ps=2048), dict(trs=9), dict(tp=0), dict(tp=1 << 27, trs=1 << 27), dict(tree=I4, words=0), dict(tree=I4, words=65),
    dict(tree=I4 + 4, words=1), dict(window=-1), dict(sinks=-1), dict(scale=-1.0), dict(scale=float("inf")),
    dict(out=Q), dict(out=KP + 256), dict(keys=(1 << 30) + 1),
    dict(B=1, keys=160000, tp=10000, trs=10000, ws=0), dict(B=1, keys=160000, tp=10000, trs=10000, wsb=256),
    dict(B=1, keys=160000, tp=10000, trs=10000, ws=KP), dict(B=1, keys=160000, tp=10000, trs=10000, ws=O),
], ids=str)
def test_attention_refuses(kw):
    assert _attend(**kw) == BAD


def _append(**kw):
    a = dict(q=Q, k=K, v=V, qrs=1024, krs=256, vrs=256, qo=O, qors=1024, kp=KP, vp=VP, ps=4096, rs=256, hs=128, n_pages=40,
             page=16, table=I1, trs=10, tp=10, starts=I2, lens=I3, pos=0, B=3, T=12, H=8, HK=2, qw=0, kw=0, kind=1, ta=I4,
             tb=I5, tabs=64, rows=100, pairing=0, rot=128, eps=1e-6, stream=None)
    a.update(kw)
    return cache.lib().lr_cache_append_bf16(*a.values())


@pytest.mark.parametrize("kw", [
    dict(k=0), dict(v=0), dict(qo=0), dict(kp=0), dict(vp=0), dict(table=0), dict(starts=0), dict(lens=0), dict(T=0),
    dict(H=0), dict(HK=0), dict(B=0), dict(qrs=1020), dict(krs=128), dict(qors=512), dict(page=24), dict(n_pages=0),
    dict(qw=I6 + 4), dict(kw=I6 + 8), dict(kind=9), dict(ta=0), dict(tb=0), dict(tabs=63), dict(rows=0), dict(pairing=2),
    dict(rot=130), dict(rot=63), dict(pairing=1, rot=40), dict(eps=-1.0), dict(eps=float("nan")), dict(pos=I6 + 2),
    dict(qo=Q + 256), dict(qo=Q, qors=2048), dict(k=KP), dict(v=VP + 4096), dict(q=KP), dict(qo=VP), dict(qo=K),
], ids=str)
def test_append_refuses(kw):
    assert _append(**kw) == BAD


# in place on rows of 8 query heads: k or v over columns that are overwritten
@pytest.mark.parametrize("kw", [
    dict(k=Q), dict(v=Q), dict(k=Q + 2 * 896), dict(v=Q + 2 * (1536 - 128)), dict(k=Q + 2 * (5 * 1536 + 512)),
    dict(v=Q + 2 * (1016)), dict(k=Q - 2 * 128), dict(k=Q + 2 * 1024, krs=768), dict(v=Q + 2 * 1024, vrs=1584),
    dict(k=Q, krs=256, T=1), dict(v=Q + 2 * 1000, vrs=256, T=1),
], ids=str)
def test_append_in_place_refuses_keys_and_values_in_the_queries_columns(kw):
    assert _append(**dict(dict(qo=Q, qrs=1536, qors=1536, krs=1536, vrs=1536), **kw)) == BAD


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses of calls that are not refused are no memory")
@pytest.mark.parametrize("kw", [
    dict(), dict(k=Q + 2 * 1024, v=Q + 2 * 1280), dict(k=Q + 2 * (4 * 1536 + 1024)), dict(v=Q + 2 * (1280 - 1536)),
    dict(v=Q + 2 * 1024, vrs=1552),   # (row u, from column 1024 + 16 u on, ends at column 1456 at most)
    dict(k=Q + 2 * 1024, krs=4608), dict(k=Q + 2 * 1024, krs=256, T=1), dict(k=Q + 2 * (1024 + 11 * 1536), krs=256),
], ids=str)
def test_append_in_place_on_a_packed_projection(kw):
    """Keys and values in columns of their own, of these rows or others, are none of the queries' (without a GPU such a call ends in
    an error of its own)."""
    assert _append(**dict(dict(qo=Q, qrs=1536, qors=1536, krs=1536, vrs=1536), **kw)) != BAD


def _copy(**kw):
    a = dict(kp=KP, vp=VP, layers=2, ls=1 << 20, ps=4096, rs=256, hs=128, n_pages=40, page=16, HK=2, src=I1, dst=I2, n=5,
             stream=None)
    a.update(kw)
    return cache.lib().lr_cache_copy_pages(*a.values())


def _move(**kw):
    a = dict(kp=KP, vp=VP, layers=2, ls=1 << 20, ps=4096, rs=256, hs=128, n_pages=40, page=16, HK=2, table=I1, trs=10, tp=10,
             starts=I2, src=I3, dst=I4, B=3, n=9, rows=5, stream=None)
    a.update(kw)
    return cache.lib().lr_cache_move_rows(*a.values())


@pytest.mark.parametrize("kw", [dict(kp=0), dict(vp=0), dict(layers=0), dict(ls=4), dict(ls=-8), dict(ps=100), dict(page=3),
                                dict(HK=0), dict(src=0), dict(dst=0), dict(dst=I2 + 2), dict(n=0), dict(n=-1)], ids=str)
def test_copy_refuses(kw):
    assert _copy(**kw) == BAD


@pytest.mark.parametrize("kw", [dict(kp=0), dict(vp=0), dict(layers=0), dict(layers=40000), dict(ls=-8), dict(rs=100),
                                dict(page=3), dict(table=0), dict(starts=0), dict(src=0), dict(dst=0), dict(B=0), dict(n=0),
                                dict(rows=0), dict(rows=257), dict(trs=9)], ids=str)
def test_move_refuses(kw):
    assert _move(**kw) == BAD


def test_pools_that_share_rows_are_refused():
    """Keys and values may interleave in one buffer (rows of their own), but not share rows; layers neither."""
    assert _attend(vp=KP) == _append(vp=KP) == _copy(vp=KP) == _move(vp=KP) == BAD
    assert _attend(vp=KP + 128) == _append(vp=KP - 240) == BAD
    for ls in (0, 64):
        assert _copy(ls=ls) == _move(ls=ls) == BAD


def _rows_of(base, layers, ls, ps, rs, hs, n_pages, page, HK):
    """(set of the pool's heads' rows in units of 8 elements, their number) of one of keys and values."""
    units = [base + l * ls + p * ps + r * rs + h * hs + x for l in range(layers) for p in range(n_pages) for r in range(page)
             for h in range(HK) for x in range(0, 128, 8)]
    return set(units), len(units)


def _shares(d, **kw):
    k, nk = _rows_of(0, **kw)
    v, _ = _rows_of(d, **kw)
    return len(k) < nk or bool(k & v)


PARTLY = [   # keys' rows and values' rows d elements apart; layers, their stride, strides of pages, rows and heads
    dict(d=128, layers=1, ls=0, ps=4096, rs=256, hs=128),            # value head 0 is key head 1
    dict(d=-128, layers=1, ls=0, ps=4096, rs=256, hs=128),
    dict(d=8, layers=1, ls=0, ps=4096, rs=256, hs=128),
    dict(d=4096, layers=1, ls=0, ps=4096, rs=256, hs=128),           # value page 0 is key page 1
    dict(d=4096 - 256, layers=1, ls=0, ps=4096, rs=256, hs=128),     # value row 0 is the last key row of page 0
    dict(d=39 * 4096 + 15 * 256 + 128, layers=1, ls=0, ps=4096, rs=256, hs=128),   # the last row alone
    dict(d=256 - 64, layers=1, ls=0, ps=8192, rs=512, hs=128),       # half a head
    dict(d=1 << 40, layers=2, ls=128, ps=4096, rs=256, hs=128),      # layer 1's head 0 is layer 0's head 1
    dict(d=1 << 40, layers=2, ls=4096, ps=4096, rs=256, hs=128),     # layer 1's page 0 is layer 0's page 1
    dict(d=1 << 40, layers=3, ls=39 * 4096 + 8, ps=4096, rs=256, hs=128),
    dict(d=256, layers=5, ls=64 * 4096, ps=8192, rs=512, hs=128, n_pages=33),      # the layers meet, keys and values do not
    dict(d=4 << 20, layers=3, ls=2 << 20, ps=4096, rs=256, hs=128),  # layer 0's values are layer 2's keys
]


@pytest.mark.parametrize("c", PARTLY, ids=lambda c: "-".join(map(str, c.values())))
def test_pools_that_share_some_rows_are_refused(c):
    a = dict(dict(n_pages=40, page=16, HK=2), **c)
    assert _shares(**a)
    kw = {x: a[x] for x in ("layers", "ls", "ps", "rs", "hs", "n_pages")}
    kp = 1 << 44
    assert _copy(kp=kp, vp=kp + 2 * a["d"], **kw) == _move(kp=kp, vp=kp + 2 * a["d"], **kw) == BAD
    if a["layers"] == 1:
        one = {x: a[x] for x in ("ps", "rs", "hs", "n_pages")}
        assert _attend(kp=kp, vp=kp + 2 * a["d"], **one) == _append(kp=kp, vp=kp + 2 * a["d"], **one) == BAD


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses of calls that are not refused are no memory")
def test_pools_are_refused_where_they_share_rows_and_nowhere_else():
    """Random small layouts, nested in every order and not nested, against the rows themselves. (Without a GPU a call that is not
    refused ends in an error of its own.)"""
    rng = random.Random(3)
    some = [0, 0]
    for _ in range(1500):
        layers, n_pages, page, HK = rng.choice([1, 2, 3, 5]), rng.choice([1, 2, 4]), rng.choice([1, 2, 4]), rng.choice([1, 2, 3])
        dims = [["ls", layers], ["ps", n_pages], ["rs", page], ["hs", HK], ["kv", 2]]
        rng.shuffle(dims)
        at, st = 128, {}
        for name, n in dims:
            st[name] = at
            at = at * n + rng.choice([0, 0, 0, 8, 128])
        if rng.random() < 0.5:
            st["kv"] = rng.choice([1, -1]) * 8 * rng.randrange(0, at // 8 + 2)
        if rng.random() < 0.3:
            st["ls"] = 8 * rng.randrange(16, at // 8 + 2)
        kw = dict(layers=layers, ls=st["ls"], ps=st["ps"], rs=st["rs"], hs=st["hs"], n_pages=n_pages, page=page, HK=HK)
        token = st["rs"] >= (HK - 1) * st["hs"] + 128 and st["ps"] >= (page - 1) * st["rs"] + (HK - 1) * st["hs"] + 128
        head = st["hs"] >= (page - 1) * st["rs"] + 128 and st["ps"] >= (HK - 1) * st["hs"] + (page - 1) * st["rs"] + 128
        if not token and not head:
            continue
        shared = _shares(st["kv"], **kw)
        some[shared] += 1
        kp = 1 << 44
        assert (_copy(kp=kp, vp=kp + 2 * st["kv"], **kw) == BAD) == shared, (kw, st["kv"])
    assert min(some) > 100


def test_parts_past_32_bits_are_refused():
    """A block's parts are addressed in 32 bits: 2^30 keys in pages of one row would have more (a launch error, not a kernel)."""
    assert cache.attention_ws_bytes(1, 1, 1, 1 << 30, 1, 1, 1) > 1 << 31
    assert _attend(B=1, T=1, rows=1, keys=1 << 30, H=1, HK=1, page=1, tp=1 << 30, trs=1 << 30, qrs=128, ors=128, ps=128, rs=128,
                   wsb=1 << 40, ws=1 << 44) == BAD


@pytest.mark.parametrize("T", [524304, 524312, 524360, 1 << 24])
def test_launches_past_a_grid_are_refused(T):
    """65,535 sequences and max_rows left at all the tokens: 65,535 x 8 x 16 T / 128 blocks of rows, whose number an XCD is 65,534 or
    a little more when it is cut to 32 bits. Refused before that, not launched with too few."""
    far = dict(q=1 << 44, out=2 << 44, kp=3 << 44, vp=4 << 44, table=5 << 44, starts=6 << 44, lens=7 << 44, ws=8 << 44, wsb=1 << 43)
    assert _attend(B=65535, T=T, rows=T, keys=160, H=128, HK=8, qrs=128 * 128, ors=128 * 128, ps=16 * 1024, rs=1024, **far) == BAD


def test_python_checks_refuse_host_tensors():
    t = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    p = torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.attention_window(t, t, t, window=4)
    with pytest.raises(ValueError):
        cache.attention(t, p, p, i[None], i[:2], i[:1])
    with pytest.raises(ValueError):
        cache.append(t, t, t, p, p, i[None], i[:2], i[:1], table_kind=ops.TABLE_NONE)
    if not torch.cuda.is_available():
        with pytest.raises(ValueError):
            cache.copy_pages(p, p, i, i)
        with pytest.raises(ValueError):
            cache.move_rows(p, p, i[None], i[:2], i, i)


# ------------------------------------------------------------------------------------------------ bookkeeping
def test_pool_alloc_fork_free():
    pool = cache.PagePool(5)
    a = pool.alloc(3)
    assert len(set(a)) == 3 and pool.free_pages == 2
    with pytest.raises(MemoryError):
        pool.alloc(3)
    assert pool.free_pages == 2
    b = pool.fork(a)
    assert b == a and b is not a and pool.free_pages == 2
    pool.free(a)
    assert pool.free_pages == 2          # still held by the fork
    pool.free(b)
    assert pool.free_pages == 5
    for bad in ([a[0]], [-1], [5]):
        with pytest.raises(ValueError):
            pool.free(bad)
    c = pool.alloc(1)
    with pytest.raises(ValueError):
        pool.free(c + c)                 # once held, freed twice in one call: nothing happens
    assert pool.free_pages == 4 and pool.alloc(0) == []


def test_pool_own_gives_a_page_of_its_own():
    pool = cache.PagePool(4)
    a = pool.alloc(2)
    assert pool.own(a, 1) is None
    b = pool.fork(a)
    src, dst = pool.own(b, 1)
    assert src == a[1] and dst == b[1] and dst not in a and b[0] == a[0]
    assert pool.own(a, 1) is None and pool.own(b, 1) is None     # each its own now
    pool.free(a)
    pool.free(b)
    assert pool.free_pages == 4


def test_pool_compact_packs_to_the_front():
    pool = cache.PagePool(8)
    a, b, c = pool.alloc(3), pool.alloc(2), pool.alloc(2)
    d = pool.fork(c)
    pool.free(a)
    with pytest.raises(ValueError):
        pool.compact([b, c])             # the fork's table is missing
    tables = [b, c, d]
    before = [list(t) for t in tables]
    src, dst = pool.compact(tables)
    assert not set(src) & set(dst) and all(x >= 4 for x in src) and all(x < 4 for x in dst)
    moved = dict(zip(src, dst))
    assert tables == [[moved.get(p, p) for p in t] for t in before] and sorted({p for t in tables for p in t}) == [0, 1, 2, 3]
    assert c == d and pool.free_pages == 4 and sorted(pool.alloc(4)) == [4, 5, 6, 7]
    assert pool.compact([]) == ([], []) if pool.free_pages == 8 else True


def test_pool_compact_of_nothing():
    for pool in (cache.PagePool(8), cache.PagePool(1)):
        n = pool.free_pages
        assert pool.compact([]) == ([], []) and pool.free_pages == n and sorted(pool.alloc(n)) == list(range(n))
    pool = cache.PagePool(8)
    pool.free(pool.alloc(5))
    assert pool.compact([[], []]) == ([], []) and pool.free_pages == 8
    pool.alloc(1)
    with pytest.raises(ValueError):
        pool.compact([])


def test_host_calls_refuse_host_tensors_by_name():
    """The calls' own checks, past the Python side's: every tensor is refused by its name, with what it is."""
    h = cache._host()
    t = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    p = torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match=r"q: expected bf16 \[4, 2, 128\].*BFloat16 \[4, 2, 128\] / \[256, 128, 1\] on cpu"):
        h.attention(-1, 0, t, p, p, i[None], i, i[:1], None, None, None, None, 0, 0, 0.1, None)
    with pytest.raises(ValueError, match="k_pages, v_pages"):
        h.append(-1, 0, t, t, t, p, p, i[None], i, i[:1], None, None, None, 0, None, None, None, 0, 128, 1e-6)
    with pytest.raises(ValueError, match="k_pages, v_pages: expected .* or .layers"):
        h.copy_pages(-1, 0, p, p, i, i)
    with pytest.raises(ValueError, match="k_pages: expected a tensor on the current device, got NoneType"):
        h.move_rows(-1, 0, None, p, i[None], i, i, i, None)
    with pytest.raises(ValueError, match="q: expected bf16"):
        h.attention_window(-1, 0, t, t, t, None, 4, 0, 1, 0, 0.1, None)
    with pytest.raises(TypeError):
        h.attention(1, 2, 3)
    with pytest.raises(TypeError):
        h.attention("cuda", 0, t, p, p, i[None], i, i[:1], None, None, None, None, 0, 0, 0.1, None)


@pytest.mark.parametrize("kind,rot,columns", [(ops.TABLE_COSSIN_F32, 128, 64), (ops.TABLE_COSSIN_F32, 0, 64), (ops.TABLE_COSSIN_F32, 96, 48),
                                              (ops.TABLE_MAT2_BF16, 128, 256), (ops.TABLE_MAT2_F32, 64, 128)])
def test_append_refuses_tables_that_are_narrower_than_the_rotation(kind, rot, columns):
    """A view of a table's columns has its parent's row stride: with fewer columns than the rotation takes, a row would go on in the
    next one and the last row past the storage."""
    h = cache._host()
    x, p, i = torch.zeros(4, 2, 128, dtype=torch.bfloat16), torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int32)
    whole = torch.zeros(50, 2 * columns, dtype=torch.bfloat16 if kind == ops.TABLE_MAT2_BF16 else torch.float32)
    call = lambda a, b: h.append(-1, 0, None, x, x, p, p, i[None], i, i[:1], None, None, None, kind, a, b, None, 0, rot, 1e-6)
    two = kind == ops.TABLE_COSSIN_F32
    for a, b in ((whole[:, columns + 1:], whole[:, columns + 1:]), (whole[:, :columns - 1], whole[:, :columns - 1]),
                 (whole[:, :columns], whole[:, :columns - 1])):
        if two or a.shape[1] < columns:
            with pytest.raises(ValueError, match=rf"table: rows of {columns - 1} columns, rot {rot} needs {columns}"):
                call(a, b if two else None)
    # wide enough (the next refusal is the host tensors'), and no table at all
    for a in (whole, whole[:, :columns], whole[:, columns:]):
        with pytest.raises(ValueError, match="k_pages, v_pages"):
            call(a, a if two else None)
    with pytest.raises(ValueError, match="table: expected a tensor"):
        call(None, None)


@pytest.mark.parametrize("missing", ["torch", "Python.h"])
def test_the_library_is_built_without_torch_or_python_headers(missing, monkeypatch, tmp_path, capsys):
    """The extension is left out and said to be, an older one goes away, and nothing else fails."""
    import importlib.util
    import sysconfig

    from localrouter_amd import build
    find, paths = importlib.util.find_spec, sysconfig.get_paths()
    if missing == "torch":
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    else:
        monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **kw: dict(paths, include=str(tmp_path)))
    old = tmp_path / "_host_calls.so"
    old.write_bytes(b"old")
    monkeypatch.setattr(build, "HOST_CALLS_LIB", old)
    monkeypatch.setattr(build, "_run", lambda cmd: pytest.fail(f"ran {cmd}"))
    assert build.build_host_calls() is None and not old.exists()
    assert "without localrouter_amd.cache's host calls" in capsys.readouterr().err


def test_calls_without_the_extension_raise(monkeypatch):
    import sys

    import localrouter_amd
    monkeypatch.setitem(sys.modules, "localrouter_amd._host_calls", None)
    monkeypatch.delattr(localrouter_amd, "_host_calls", raising=False)
    monkeypatch.setattr(cache, "_calls", None)
    with pytest.raises(RuntimeError, match="_host_calls is missing"):
        cache._host()
