"""Attention over prompts packed end to end (ops.attention_packed) against a 64-bit attention over exactly the seen keys."""
from __future__ import annotations

import pytest
import torch

from localrouter_amd import _lib, cache, ops
from tests.cache_util import check_rows, gen, ref_rows, rnd

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def sums(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def seen_of(n, window=0, sinks=0):
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    return (j <= i) & ((i - j < window) | (j < sinks) if window else torch.ones(1, dtype=torch.bool))


def some(n, most=40):
    """All tokens of a short sequence, the first, last and those beside tiles' borders of a long one."""
    if n <= most:
        return list(range(n))
    return sorted({i for i in (0, 1, 31, 32, 63, 64, 127, 128, n // 2, n - 65, n - 64, n - 33, n - 2, n - 1) if 0 <= i < n})


def check(q, k, v, out, lens, window=0, sinks=0, scale=1.0 / 128 ** 0.5, most=40):
    st = sums(lens)
    for b, n in enumerate(lens):
        if n:
            at = some(n, most)
            rows = [st[b] + i for i in at]
            s = slice(st[b], st[b] + n)
            check_rows(out[rows], *ref_rows(q[rows], k[s], v[s], seen_of(n, window, sinks)[at], scale), what=f"sequence {b}")


# lengths, heads, kv heads, window, sinks
CASES = [
    ([1], 1, 1, 0, 0),
    ([1], 8, 2, 0, 0),
    ([2, 1, 3], 4, 4, 0, 0),
    ([17, 0, 16, 1, 15], 4, 1, 0, 0),                # a sequence without tokens
    ([33, 32, 31, 64, 65], 2, 2, 0, 0),
    ([100, 5, 300], 7, 1, 0, 0),
    ([513], 3, 3, 0, 0),
    ([200, 1, 700, 90], 8, 2, 0, 0),
    ([200, 1, 700, 90], 8, 2, 50, 0),
    ([200, 1, 700, 90], 8, 2, 33, 5),
    ([1500, 20], 16, 16, 0, 0),
    ([1100, 700, 64, 128], 32, 8, 0, 0),
    ([1100, 700, 64, 128], 32, 8, 64, 65),
    ([2500, 1], 64, 8, 0, 0),
    ([2500, 1], 64, 8, 1, 0),                        # a window of the token itself
    ([130] * 30, 24, 8, 0, 0),
    ([1 + 7 * i % 50 for i in range(64)], 6, 2, 0, 0),
    ([1 + 7 * i % 50 for i in range(65)], 6, 2, 0, 0),             # more sequences than lanes
    ([(i * 37) % 90 for i in range(200)], 16, 8, 0, 0),
    ([(i * 37) % 90 for i in range(200)], 32, 8, 20, 3),
    ([0] * 300 + [400], 40, 8, 0, 0),
    ([3000, 2000], 64, 4, 0, 0),
]


def _ids(c):
    return f"{len(c[0])}seq{max(c[0])}h{c[1]}g{c[2]}w{c[3]}s{c[4]}"


@pytest.mark.parametrize("c", CASES, ids=_ids)
def test_packed_matches_64_bits(c):
    lens, H, HK, window, sinks = c
    g, T = gen(7 + len(lens)), sum(lens)
    q, k, v = rnd(g, T, H, 128), rnd(g, T, HK, 128), rnd(g, T, HK, 128)
    out = ops.attention_packed(q, k, v, ints(sums(lens)), window=window, sinks=sinks)
    check(q, k, v, out, lens, window, sinks)


@pytest.mark.parametrize("c", CASES, ids=_ids)
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_views_paddings_and_rows_of_no_sequence(c, what):
    """Views of one packed projection, an output with wider rows; rows before the first sequence and behind the last hold NaN or
    infinities, and their output rows stay as they were."""
    lens, H, HK, window, sinks = c
    lead, tail = 5, 70
    T = lead + sum(lens) + tail
    g = gen(9 + len(lens))
    qkv = rnd(g, T, H + 2 * HK, 128)
    qkv[:lead], qkv[T - tail:] = what, what
    q, k, v = qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:]
    wide = torch.full((T, H + 1, 128), 5.0, dtype=BF16, device="cuda")
    st = [lead + x for x in sums(lens)]
    ops.attention_packed(q, k, v, ints(st), wide[:, 1:], window=window, sinks=sinks)
    assert (wide[:lead] == 5.0).all() and (wide[T - tail:] == 5.0).all() and (wide[:, 0] == 5.0).all()
    s = slice(lead, T - tail)
    check(q[s], k[s], v[s], wide[s, 1:], lens, window, sinks, most=3)


@pytest.mark.parametrize("heads", [(4, 2), (64, 8), (96, 32)])
def test_later_tokens_have_no_part(heads):
    """An infinity or NaN in a later token, or in another sequence, stays there; in a seen one it shows."""
    H, HK = heads
    lens = [90, 300, 40]
    T = sum(lens)
    g = gen(11)
    q, k, v = rnd(g, T, H, 128), rnd(g, T, HK, 128), rnd(g, T, HK, 128)
    k[90 + 200], v[90 + 250] = float("nan"), float("inf")
    out = ops.attention_packed(q, k, v, ints(sums(lens)))
    assert torch.isfinite(out[:90 + 200]).all() and torch.isfinite(out[390:]).all()
    assert out[290:390].isnan().all()
    check(q, k, v, out, lens)


@pytest.mark.parametrize("scale", [0.02, 1.0])
@pytest.mark.parametrize("H", [2, 97])
def test_large_scores(scale, H):
    """Scores far from zero, rising along the keys, so that the references are raised again and again."""
    g = gen(13)
    lens = [700, 90]
    q, k, v = rnd(g, 790, H, 128), rnd(g, 790, H, 128), rnd(g, 790, H, 128)
    k = (k.float() * torch.linspace(0.1, 2.0, 790, device="cuda")[:, None, None]).to(BF16)
    out = ops.attention_packed(q, k, v, ints(sums(lens)), scale=scale)
    at = sorted({0, 1, H - 1})
    check(q[:, at], k[:, at], v[:, at], out[:, at], lens, scale=scale)


@pytest.mark.parametrize("H,HK", [(4, 2), (32, 8)])
def test_one_sequence_is_causal_attention(H, HK):
    g = gen(15)
    q, k, v = rnd(g, 777, H, 128), rnd(g, 777, HK, 128), rnd(g, 777, HK, 128)
    a = ops.attention_packed(q, k, v, ints([0, 777])).double().cpu()
    b = ops.attention(q, k, v, causal=True).double().cpu()
    at = some(777)
    _, mag = ref_rows(q[at], k, v, seen_of(777)[at])
    # both round P and the output to bf16: each is within the tolerance of the other's exact value
    assert ((a - b).abs()[at] <= 2 * (2.0 ** -8 * b.abs()[at] + (2.0 ** -7 + 2.0 ** -10) * mag)).all()


@pytest.mark.parametrize("starts", [[0, 50, 20, 100], [-7, 20, 60, 100], [0, 30, 60, 1 << 30], [0, 0, 0, 0], [100, 100, 100, 100],
                                    [5, 4, 3, 2], [-(1 << 31), 0, (1 << 31) - 1, 9], [40, 101, 50, 100]])
@pytest.mark.parametrize("H,B", [(4, 3), (64, 3), (64, 90), (512, 3), (512, 90)])
def test_senseless_starts_touch_nothing_outside(starts, H, B):
    """Starts that do not ascend or lie outside: whatever rows come out, nothing outside the output's rows is written."""
    g = gen(17)
    q, k, v = rnd(g, 100, H, 128), rnd(g, 100, 4, 128), rnd(g, 100, 4, 128)
    out = torch.full((104, H, 128), 5.0, dtype=BF16, device="cuda")
    st = starts + [starts[-1]] * (B - 3)
    ops.attention_packed(q, k, v, ints(st), out[2:102])
    assert (out[:2] == 5.0).all() and (out[102:] == 5.0).all()


@pytest.mark.parametrize("H,HK", [(8, 2), (32, 8), (64, 8)])
def test_captured_and_replayed(H, HK):
    """A captured call follows starts and the rows at its replay; bit for bit the eager call's; on a stream of its own."""
    T, g = 900, gen(19)
    q, k, v = rnd(g, T, H, 128), rnd(g, T, HK, 128), rnd(g, T, HK, 128)
    st, out = ints([0, 300, 301, 800]), torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.attention_packed(q, k, v, st, out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_packed(q, k, v, st, out)
    for lens in ([900, 0, 0], [1, 2, 3], [300, 300, 300], [0, 899, 1]):
        st.copy_(ints(sums(lens)))
        for t in (q, k, v):
            t.copy_(rnd(g, *t.shape))
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert (got[sum(lens):] == 3.0).all()
        ops.attention_packed(q, k, v, st, out)
        assert torch.equal(got, out)
        check(q, k, v, got, lens, most=3)


def test_far_rows():
    """Rows whose offsets pass 32 bits."""
    H, n = 2, 700
    big = torch.zeros(n, 1 << 22, dtype=BF16, device="cuda")
    k, v = (big[:, i * 256:i * 256 + 256].view(n, 2, 128) for i in (0, 1))
    g = gen(23)
    k.copy_(rnd(g, n, 2, 128))
    v.copy_(rnd(g, n, 2, 128))
    for heads in (H, 64):
        q = rnd(g, n, heads, 128)
        lens = [100, 600]
        out = ops.attention_packed(q, k, v, ints(sums(lens)))
        check(q, k, v, out, lens)


def test_prompts_into_a_cache():
    """Prompts through packed attention, their keys and values appended to pages of bf16 and of 8 bits: the next tokens' attention over
    the pages continues them."""
    from tests.cache8_util import E8, F8, values
    from tests.test_gpu_cache import chain_seen
    lens, H, HK, ps = [70, 33, 1], 8, 2, 16
    T, g, st = sum(lens), gen(29), sums(lens)
    table = ints([[0, 2, 4, 6, 8], [1, 3, 5, -1, -1], [7, -1, -1, -1, -1]])
    kp, vp = (torch.zeros(9, ps, HK, 128, dtype=BF16, device="cuda") for _ in range(2))
    k8, v8 = (torch.zeros(9, ps, HK, 128, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2))
    ks, vs = (torch.zeros(9, 1, HK, dtype=torch.uint8, device="cuda").view(E8) for _ in range(2))
    a = torch.arange(80, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    tab = (a.cos().float().cuda(), a.sin().float().cuda())
    q, k, v = rnd(g, T, H, 128), rnd(g, T, HK, 128), rnd(g, T, HK, 128)
    qo = cache.append(q, k, v, kp, vp, table, ints(st), ints(lens), table=tab)
    assert torch.equal(qo, cache.append_f8(q, k, v, k8, v8, ks, vs, table, ints(st), ints(lens), table=tab))
    rows = lambda p, b, n: p[table[b][torch.arange(n, device="cuda") // ps].long(), torch.arange(n, device="cuda") % ps]
    kr = torch.cat([rows(kp, b, n) for b, n in enumerate(lens)])   # (rotated)
    out = ops.attention_packed(qo, kr, v, ints(st))
    check(qo, kr, v, out, lens)
    over = cache.attention(qo, kp, vp, table, ints(st), ints(lens), max_rows=70, max_keys=70)
    check(qo, kr, v, over, lens)
    nxt = [n + 1 for n in lens]
    q, k, v = rnd(g, 3, H, 128), rnd(g, 3, HK, 128), rnd(g, 3, HK, 128)
    qo = cache.append_f8(q, k, v, k8, v8, ks, vs, table, ints([0, 1, 2, 3]), ints(nxt), table=tab)
    out = cache.attention_f8(qo, k8, v8, ks, vs, table, ints([0, 1, 2, 3]), ints(nxt), max_rows=1, max_keys=80)
    for b, n in enumerate(nxt):
        check_rows(out[b:b + 1], *ref_rows(qo[b:b + 1], rows(values(k8, ks), b, n), rows(values(v8, vs), b, n), chain_seen(1, n)))


def test_refusals_by_name():
    q, k = torch.zeros(4, 4, 128, dtype=BF16, device="cuda"), torch.zeros(4, 2, 128, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="different lengths"):
        ops.attention_packed(q[:3], k, k, ints([0, 3]))
    with pytest.raises(ValueError, match="starts"):
        ops.attention_packed(q, k, k, ints([0]))
    with pytest.raises(ValueError, match="starts"):
        ops.attention_packed(q, k, k, ints([0, 4]).long())
    with pytest.raises(ValueError, match="bf16"):
        ops.attention_packed(q.float(), k, k, ints([0, 4]))
    with pytest.raises(_lib.LrError):
        ops.attention_packed(q, k, k, ints([0, 4]), q)
    assert ops.attention_packed(q[:0], k[:0], k[:0], ints([0, 0])).shape == (0, 4, 128)
