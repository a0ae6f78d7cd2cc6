"""The windowed attention (ops.attention_window) against a 64-bit attention over exactly the seen keys."""
from __future__ import annotations

import pytest
import torch

from localrouter_amd import _lib, ops
from tests.cache_util import check_rows, gen, ref_rows, rnd, window_seen

pytestmark = pytest.mark.gpu

# queries, keys, p0, heads, kv heads, window, sinks, frame
CASES = [
    (1, 1, 0, 1, 1, 1, 0, 1),
    (1, 1, 0, 4, 1, 7, 3, 1),
    (1, 500, 499, 8, 2, 64, 4, 1),
    (1, 3000, 2999, 4, 4, 3000, 0, 1),            # split over the keys
    (1, 9000, 8999, 7, 1, 5000, 33, 1),           # split, seven heads over one
    (2, 65, 63, 4, 2, 1, 0, 1),                   # a window of the token itself
    (33, 33, 0, 2, 2, 8, 1, 1),
    (64, 200, 136, 4, 1, 31, 32, 1),
    (77, 411, 300, 6, 2, 100, 65, 1),             # queries past the last key
    (130, 130, 0, 3, 1, 1000, 0, 1),              # a window wider than the keys: causal
    (200, 150, 0, 2, 1, 40, 2, 1),                # more queries than keys
    (5, 100, 180, 2, 1, 20, 0, 1),                # nothing to see: every key lies before the window
    (5, 100, 118, 2, 1, 20, 0, 1),                # the first queries see one key, the later ones none
    (5, 100, 180, 2, 1, 20, 3, 1),                # only the first tokens
    (300, 700, 400, 8, 8, 64, 4, 1),
    (96, 96, 0, 2, 1, 2, 0, 32),                  # frames of a tile
    (190, 190, 0, 2, 2, 2, 10, 50),               # frames that end inside tiles
    (70, 190, 120, 2, 2, 1, 0, 50),               # a chunk that starts inside a frame, keys that end inside one
    (257, 1025, 768, 4, 2, 3, 77, 100),
    (13, 2000, 1700, 5, 5, 2, 100, 1000),
    (640, 640, 0, 1, 1, 1 << 30, 1 << 30, 1 << 30),   # one frame: every query sees every key
]


def _ids(c):
    return "x".join(map(str, c))


@pytest.mark.parametrize("c", CASES, ids=_ids)
def test_window_matches_64_bits(c):
    w, n, p0, H, HK, window, sinks, frame = c
    g = gen(7 + w + n)
    q, k, v = rnd(g, w, H, 128), rnd(g, n, HK, 128), rnd(g, n, HK, 128)
    out = ops.attention_window(q, k, v, window=window, sinks=sinks, frame=frame, p0=p0)
    check_rows(out, *ref_rows(q, k, v, window_seen(w, n, p0, window, sinks, frame)))


@pytest.mark.parametrize("frame,window,sinks", [(1, 4100, 5), (500, 9, 700)])
def test_window_of_whole_rounds(frame, window, sinks):
    """Enough blocks and keys for the workgroups of eight waves: 1,024 queries x 64 heads over 8; some queries checked."""
    g = gen(21)
    q, k, v = rnd(g, 1024, 64, 128), rnd(g, 5500, 8, 128), rnd(g, 5500, 8, 128)
    out = ops.attention_window(q, k, v, window=window, sinks=sinks, frame=frame, p0=4400)
    at = [0, 1, 31, 32, 33, 63, 64, 99, 100, 511, 600, 1022, 1023]
    check_rows(out[at], *ref_rows(q[at], k, v, window_seen(1024, 5500, 4400, window, sinks, frame)[at]))


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_window_scale_and_large_scores(scale):
    """Scores far from zero, rising along the keys, so that the reference of every row is raised again and again."""
    g = gen(3)
    q, k, v = rnd(g, 100, 2, 128), rnd(g, 900, 2, 128), rnd(g, 900, 2, 128)
    k = (k.float() * torch.linspace(0.1, 2.0, 900, device="cuda")[:, None, None]).to(torch.bfloat16)
    out = ops.attention_window(q, k, v, window=500, sinks=3, p0=800, scale=scale)
    check_rows(out, *ref_rows(q, k, v, window_seen(100, 900, 800, 500, 3, 1), scale))


@pytest.mark.parametrize("c", [c for c in CASES if c[0] * c[3] // c[4] > 64], ids=_ids)
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_window_of_many_heads(c, what):
    """So many heads that the blocks fill more than a round of the CUs, whatever the queries; the first and the last kv heads
    checked. Views of packed rows, and infinities and NaN in every key that no query sees."""
    w, n, p0, H, HK, window, sinks, frame = c
    G, many = H // HK, 96 + w % 2
    g = gen(30 + w + n)
    q, kv = rnd(g, w, G * many, 128), rnd(g, n, 2 * many + 1, 128)
    k, v = kv[:, :many], kv[:, many:2 * many]
    seen = window_seen(w, n, p0, window, sinks, frame)
    kv[~seen.any(0).cuda()] = what
    out = ops.attention_window(q, k, v, window=window, sinks=sinks, frame=frame, p0=p0)
    assert torch.isfinite(out).all()
    for hk in (0, many - 1):
        s = slice(G * hk, G * hk + G)
        check_rows(out[:, s], *ref_rows(q[:, s], k[:, hk:hk + 1], v[:, hk:hk + 1], seen), what=f"kv head {hk}")


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_window_of_many_heads_and_large_scores(scale):
    """Scores rising along the keys, past what the first reference allows for; a NaN in a seen key of one head."""
    g = gen(31)
    q, k, v = rnd(g, 100, 97, 128), rnd(g, 900, 97, 128), rnd(g, 900, 97, 128)
    k = (k.float() * torch.linspace(0.1, 2.0, 900, device="cuda")[:, None, None]).to(torch.bfloat16)
    k[850, 5, 77] = float("nan")
    out = ops.attention_window(q, k, v, window=500, sinks=3, p0=800, scale=scale)
    at = [0, 5, 50, 96]
    check_rows(out[:, at], *ref_rows(q[:, at], k[:, at], v[:, at], window_seen(100, 900, 800, 500, 3, 1), scale))


def test_wide_window_is_causal_attention():
    g = gen(4)
    q, k, v = rnd(g, 250, 8, 128), rnd(g, 700, 2, 128), rnd(g, 700, 2, 128)
    a = ops.attention_window(q, k, v, window=1 << 20, p0=450).double()
    b = ops.attention(q, k, v, causal=True, p0=450).double()
    # both round P and the output to bf16: each is within the tolerance of the other's exact value
    _, mag = ref_rows(q, k, v, window_seen(250, 700, 450, 1 << 20, 0, 1))
    assert ((a - b).abs().cpu() <= 2 * (2.0 ** -8 * b.abs().cpu() + (2.0 ** -7 + 2.0 ** -10) * mag)).all()


@pytest.mark.parametrize("w,n,p0", [(1, 4000, 3999), (40, 600, 560), (300, 900, 600)])
def test_window_strides(w, n, p0):
    """Queries, keys and values as views of packed rows, k and v of different strides, an output with wider rows whose other
    columns and rows stay as they were."""
    H, HK = 6, 3
    g = gen(5)
    qx, kx, vx = rnd(g, w, H + 5, 128), rnd(g, n, 2 * HK, 128), rnd(g, n, HK, 128)
    q, k = qx[:, 2:2 + H], kx[:, HK:]
    wide = torch.full((w + 2, H + 3, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    out = wide[1:1 + w, 1:1 + H]
    got = ops.attention_window(q, k, vx, out, window=2000, sinks=9, p0=p0)
    assert got is out
    check_rows(out, *ref_rows(q, k, vx, window_seen(w, n, p0, 2000, 9, 1)))
    rest = wide.clone()
    rest[1:1 + w, 1:1 + H] = 5.0
    assert (rest == 5.0).all()


@pytest.mark.parametrize("w,n,p0,window,sinks", [(1, 3000, 2500, 700, 5), (50, 300, 200, 60, 5), (300, 800, 400, 128, 5)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_keys_that_are_not_seen_have_no_part(w, n, p0, window, sinks, what):
    """Infinities and NaN in every key and value that no query sees, and in some that only a few see."""
    g = gen(6)
    q, k, v = rnd(g, w, 4, 128), rnd(g, n, 2, 128), rnd(g, n, 2, 128)
    seen = window_seen(w, n, p0, window, sinks, 1)
    no_one = ~seen.any(0).cuda()
    k[no_one] = what
    v[no_one] = what
    clean = ops.attention_window(q, k, v, window=window, sinks=sinks, p0=p0)
    assert torch.isfinite(clean).all()
    check_rows(clean, *ref_rows(q, k, v, seen))
    # the last query's own value: of the queries, it alone sees it
    v[p0 + w - 1, 0, 5] = what
    out = ops.attention_window(q, k, v, window=window, sinks=sinks, p0=p0)
    ref, mag = ref_rows(q, k, v, seen)
    check_rows(out, ref, mag)
    assert torch.isfinite(ref[:w - 1]).all() and not torch.isfinite(ref[w - 1]).all()


def test_window_nan_in_a_query_and_in_seen_keys():
    g = gen(8)
    q, k, v = rnd(g, 40, 4, 128), rnd(g, 200, 2, 128), rnd(g, 200, 2, 128)
    q[7, 1, 3] = float("nan")
    k[180, 1, 0] = float("nan")       # seen by queries at 180 .. 199 of its heads
    out = ops.attention_window(q, k, v, window=30, p0=160)
    check_rows(out, *ref_rows(q, k, v, window_seen(40, 200, 160, 30, 0, 1)))


def test_window_workspace_contents_do_not_matter():
    g = gen(9)
    q, k, v = rnd(g, 2, 8, 128), rnd(g, 6000, 2, 128), rnd(g, 6000, 2, 128)
    need = ops.attention_window_ws_bytes(2, 8, 2, 6000, window=5000, sinks=4)
    assert need > 0
    ws = torch.full((need + 512,), 255, dtype=torch.uint8, device="cuda")
    a = ops.attention_window(q, k, v, window=5000, sinks=4, p0=5998, workspace=ws)
    assert (ws[need:] == 255).all()
    b = ops.attention_window(q, k, v, window=5000, sinks=4, p0=5998)
    assert torch.equal(a, b)
    with pytest.raises(ValueError):
        ops.attention_window(q, k, v, window=5000, sinks=4, p0=5998, workspace=ws[:need - 1])


def test_window_on_other_streams_and_in_a_graph():
    """Two calls at once on streams of their own, and a captured call that follows its inputs at every replay."""
    g = gen(10)
    q, k, v = rnd(g, 3, 8, 128), rnd(g, 5000, 2, 128), rnd(g, 5000, 2, 128)
    q2 = rnd(g, 150, 8, 128)
    kw, kw2 = dict(window=3000, sinks=4, p0=4997), dict(window=300, sinks=4, p0=4850)
    want, want2 = ops.attention_window(q, k, v, **kw), ops.attention_window(q2, k, v, **kw2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s1):
            a = ops.attention_window(q, k, v, **kw)
        with torch.cuda.stream(s2):
            b = ops.attention_window(q2, k, v, **kw2)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want2)
    out = torch.empty_like(q)
    with torch.cuda.stream(s1):
        ops.attention_window(q, k, v, out, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_window(q, k, v, out, **kw)
    for seed in range(3):
        q.copy_(rnd(gen(50 + seed), 3, 8, 128))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.attention_window(q, k, v, **kw))


def test_window_rows_far_apart():
    """Row strides past what the kernel of many rows takes (2^23 elements), and offsets past 32 bits."""
    g = gen(22)
    flat = torch.zeros((1 << 23) * 300 + 4096, dtype=torch.bfloat16, device="cuda")
    k, v = flat.as_strided((300, 2, 128), (1 << 23, 128, 1)), flat.as_strided((300, 2, 128), (1 << 23, 128, 1), 1024)
    k.copy_(rnd(g, 300, 2, 128))
    v.copy_(rnd(g, 300, 2, 128))
    q = rnd(g, 50, 8, 128)
    out = ops.attention_window(q, k, v, window=100, sinks=3, p0=250)
    check_rows(out, *ref_rows(q, k, v, window_seen(50, 300, 250, 100, 3, 1)))
    near = ops.attention_window(q, k.contiguous(), v.contiguous(), window=100, sinks=3, p0=250)
    check_rows(near, *ref_rows(q, k, v, window_seen(50, 300, 250, 100, 3, 1)))
    one = ops.attention_window(q[:1], k, v, window=200, sinks=3, p0=299)
    check_rows(one, *ref_rows(q[:1], k, v, window_seen(1, 300, 299, 200, 3, 1)))
    del flat
    torch.cuda.empty_cache()


@pytest.mark.parametrize("w,H,HK,window,sinks,frame", [
    (2319, 32, 8, 2048, 4, 1),       # 64 whole blocks of an XCD before those that are cut over the keys
    (1300, 24, 12, 900, 64, 1),      # heads not by XCD, all blocks cut
    (2048, 64, 8, 5000, 0, 1),       # eight waves, two full rounds
    (2100, 64, 64, 3, 130, 700),     # frames, a last round cut
])
def test_window_of_more_rows_than_one_round(w, H, HK, window, sinks, frame):
    g = gen(24)
    n, p0 = (w + 2100, 2100) if frame == 1 else (w, 0)
    q, k, v = rnd(g, w, H, 128), rnd(g, n, HK, 128), rnd(g, n, HK, 128)
    need = ops.attention_window_ws_bytes(w, H, HK, n, window=window, sinks=sinks, frame=frame)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    out = ops.attention_window(q, k, v, window=window, sinks=sinks, frame=frame, p0=p0, workspace=ws)
    assert (ws[need:] == 255).all()
    at = torch.cat([torch.arange(0, w, 97), torch.tensor([w - 1, w - 33, w - 64])])
    seen = window_seen(w, n, p0, window, sinks, frame)[at]
    check_rows(out[at.cuda()], *ref_rows(q[at.cuda()], k, v, seen))
    assert torch.equal(out, ops.attention_window(q, k, v, window=window, sinks=sinks, frame=frame, p0=p0))


def test_window_largest_arguments():
    g = gen(23)
    q, k, v = rnd(g, 70, 2, 128), rnd(g, 150, 1, 128), rnd(g, 150, 1, 128)
    top = (1 << 31) - 1
    out = ops.attention_window(q, k, v, window=top, sinks=top, frame=top, p0=(1 << 30) - 70)
    check_rows(out, *ref_rows(q, k, v, torch.ones(70, 150, dtype=torch.bool)))
    out = ops.attention_window(q, k, v, window=top, p0=80)
    check_rows(out, *ref_rows(q, k, v, window_seen(70, 150, 80, 1 << 20, 0, 1)))


def test_window_of_no_queries():
    """As the cache's calls: an empty result, and the given tensor where there is one."""
    g = gen(12)
    q, k, v = rnd(g, 0, 4, 128), rnd(g, 9, 2, 128), rnd(g, 9, 2, 128)
    assert ops.attention_window(q, k, v, window=4).shape == (0, 4, 128)
    out = torch.full((3, 4, 128), 2.0, dtype=torch.bfloat16, device="cuda")
    assert ops.attention_window(q, k, v, out, window=4) is out and (out == 2.0).all()
    with pytest.raises(ValueError):
        ops.attention_window(q, k, v[:5], window=4)


def test_window_refuses_before_launch():
    g = gen(11)
    q, k, v = rnd(g, 4, 4, 128), rnd(g, 9, 2, 128), rnd(g, 9, 2, 128)
    for kw in (dict(window=0), dict(window=4, sinks=-1), dict(window=4, frame=0), dict(window=4, p0=-1),
               dict(window=4, scale=0.0)):
        with pytest.raises(_lib.LrError):
            ops.attention_window(q, k, v, **kw)
    with pytest.raises(_lib.LrError):
        ops.attention_window(q, k, v, q, window=4)       # in place
    with pytest.raises(ValueError):
        ops.attention_window(q.float(), k, v, window=4)
    with pytest.raises(ValueError):
        ops.attention_window(q, k, v[:5], window=4)
    with pytest.raises(ValueError):
        ops.attention_window(q, k.cpu(), v, window=4)
