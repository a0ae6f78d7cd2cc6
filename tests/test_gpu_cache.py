"""The paged cache on the GPU: attention over pages, appends, page copies and row moves, each against a plain 64-bit (or
exact) restatement, and a serving loop of them together."""
from __future__ import annotations

import random

import pytest
import torch

from localrouter_amd import _lib, cache, ops, rope
from tests.cache_util import HALF, check_rows, gen, ref_rows, rnd

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make_pool(g, pages, ps, HK, by_head=False, layers=None):
    """Two tensors [layers,] [pages, ps, HK, 128] with the same strides; by_head: rows of a head next to each other."""
    def one():
        shape = ((layers,) if layers else ()) + ((pages, HK, ps, 128) if by_head else (pages, ps, HK, 128))
        t = rnd(g, *shape)
        return t.transpose(-3, -2) if by_head else t
    return one(), one()


# empty sequences behind a batch: the launch is sized for as many blocks of rows, more than a round of the CUs, whose choice of
# kernel is another one (64 sequences of two kv heads, or more of one)
PADS = [0, 61, 300]
pads = pytest.mark.parametrize("pad", PADS)


class Batch:
    """Sequences over a pool: n tokens of the call each, L positions in all; pad: empty ones behind them."""

    def __init__(self, seed, news, lens, ps, HK, by_head=False, spare=3, pages=None, pad=0):
        news, lens = news + [0] * pad, lens + [0] * pad
        rng = random.Random(seed)
        self.g, self.ps, self.HK, self.news, self.L = gen(seed), ps, HK, news, lens
        need = [-(-x // ps) for x in lens]
        ids = list(range(pages or sum(need) + spare))
        rng.shuffle(ids)
        self.width = max(need + [1])
        self.table = []
        for n in need:
            self.table.append([ids.pop() for _ in range(n)] + [-1] * (self.width - n))
        self.n_pages = pages or sum(need) + spare
        self.kp, self.vp = make_pool(self.g, self.n_pages, ps, HK, by_head)
        self.t = ints(self.table)
        st = [0]
        for n in news:
            st.append(st[-1] + n)
        self.st, self.starts, self.lens = st, ints(st), ints(lens)

    def rows(self, b):
        """Keys and values of sequence b as rows."""
        at = torch.arange(self.L[b], device="cuda")
        page, row = self.t[b][at // self.ps].long(), at % self.ps
        return self.kp[page, row], self.vp[page, row]

    def check(self, q, out, seen_of, scale=1.0 / 128 ** 0.5):
        for b, n in enumerate(self.news):
            if n:
                k, v = self.rows(b)
                s = slice(self.st[b], self.st[b] + n)
                check_rows(out[s], *ref_rows(q[s], k, v, seen_of(b), scale), what=f"sequence {b}")


def chain_seen(n, L, window=0, sinks=0):
    p = (L - n + torch.arange(n))[:, None]
    j = torch.arange(L)[None]
    return (j <= p) & ((p - j < window) | (j < sinks) if window else torch.ones(1, dtype=torch.bool))


def random_tree(rng, n):
    sets = []
    for i in range(n):
        parent = rng.randrange(-1, i)
        sets.append({i} | (sets[parent] if parent >= 0 else set()))
    return sets


def tree_words(trees, words):
    rows = []
    for sets in trees:
        for s in sets:
            w = [sum(1 << (x & 63) for x in s if x >> 6 == u) for u in range(words)]
            rows.append([x - (1 << 64) if x >> 63 else x for x in w])
    return torch.tensor(rows, dtype=torch.int64, device="cuda")


def tree_seen(sets, L, window=0, sinks=0):
    n = len(sets)
    c = L - n
    seen = torch.zeros(n, L, dtype=torch.bool)
    for i, s in enumerate(sets):
        p = c + len(s) - 1
        for j in range(c):
            seen[i, j] = not window or p - j < window or j < sinks
        for x in s:
            seen[i, c + x] = True
    return seen


# ------------------------------------------------------------------------------------------------ attention
# tokens of each sequence, lengths, heads, kv heads, page size, window, sinks, by_head
CHAINS = [
    ([1], [1], 1, 1, 16, 0, 0, False),
    ([1], [777], 8, 2, 16, 0, 0, False),
    ([1], [5000], 4, 4, 64, 0, 0, False),                                   # split over the keys
    ([1, 1, 1], [33, 1, 400], 7, 1, 8, 0, 0, True),
    ([1, 0, 1, 1], [64, 5, 100, 31], 8, 8, 32, 0, 0, False),                # a sequence without tokens
    ([3, 1, 7], [3, 90, 7], 4, 2, 16, 0, 0, False),                         # prompts without context
    ([20, 33, 1], [220, 33, 65], 6, 2, 1, 0, 0, False),                     # pages of one row
    ([150, 9], [150, 300], 4, 1, 128, 0, 0, True),
    ([1, 1], [900, 2000], 8, 2, 16, 100, 4, False),
    ([40, 17], [300, 170], 4, 2, 4, 33, 7, False),
    ([5], [4000], 16, 1, 256, 1500, 1, True),
    ([1] * 40, [50 + 13 * i for i in range(40)], 2, 1, 16, 0, 0, False),
    ([2], [3000], 64, 1, 16, 0, 0, False),                                  # 128 rows of one kv head, split
]


@pads
@pytest.mark.parametrize("c", CHAINS, ids=lambda c: f"{len(c[0])}seq{max(c[0])}of{max(c[1])}h{c[2]}g{c[3]}p{c[4]}w{c[5]}")
def test_attention_of_chains(c, pad):
    news, lens, H, HK, ps, window, sinks, by_head = c
    B = Batch(11, news, lens, ps, HK, by_head, pad=pad)
    q = rnd(B.g, sum(news), H, 128)
    out = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, max_rows=max(news), max_keys=max(lens), window=window,
                          sinks=sinks)
    B.check(q, out, lambda b: chain_seen(news[b], lens[b], window, sinks))
    # nothing but the tensors: the table's own limits size the launch
    loose = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, window=window, sinks=sinks)
    B.check(q, loose, lambda b: chain_seen(news[b], lens[b], window, sinks))


TREES = [
    ([5], [5], 4, 2, 16, 0, 0),             # a tree and nothing before it
    ([26, 11, 1], [300, 47, 200], 8, 2, 16, 0, 0),
    ([64], [1000], 8, 1, 32, 0, 0),
    ([65, 30], [165, 63], 2, 1, 8, 0, 0),   # two words
    ([200], [330], 2, 2, 64, 0, 0),         # four words
    ([30, 8], [600, 100], 4, 1, 16, 50, 5),
    ([40], [4500], 4, 2, 16, 0, 0),         # split
]


@pads
@pytest.mark.parametrize("c", TREES, ids=lambda c: f"{len(c[0])}seq{max(c[0])}of{max(c[1])}h{c[2]}g{c[3]}p{c[4]}w{c[5]}")
def test_attention_of_trees(c, pad):
    news, lens, H, HK, ps, window, sinks = c
    rng = random.Random(5)
    trees = [random_tree(rng, n) for n in news]
    B = Batch(12, news, lens, ps, HK, pad=pad)
    q = rnd(B.g, sum(news), H, 128)
    out = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, max_rows=max(news), tree=tree_words(trees, (max(news) + 63) // 64),
                          window=window, sinks=sinks)
    B.check(q, out, lambda b: tree_seen(trees[b], lens[b], window, sinks))


@pytest.mark.parametrize("ps", [16, 64])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_whole_rounds(ps, tree):
    """Enough blocks and keys for the workgroups of eight waves: 8 sequences of 64 tokens x 128 heads over 8; the first and last
    tokens of some checked, with a page that the pool does not have."""
    news, lens = [64, 40, 64, 1, 64, 64, 50, 64], [4300, 5000, 64, 4100, 4200, 130, 4999, 2500]
    B = Batch(24, news, lens, ps, 8)
    rng = random.Random(7)
    trees = [random_tree(rng, n) for n in news]
    table = [list(r) for r in B.table]
    table[6][3] = -5
    gone = range(3 * ps, 4 * ps)
    q = rnd(B.g, sum(news), 128, 128)
    out = cache.attention(q, B.kp, B.vp, ints(table), B.starts, B.lens, max_rows=64, max_keys=5000,
                          tree=tree_words(trees, 1) if tree else None)
    for b in (0, 2, 3, 6):
        at = sorted({0, min(1, news[b] - 1), news[b] - 1})
        seen = (tree_seen(trees[b], lens[b]) if tree else chain_seen(news[b], lens[b]))[at]
        if b == 6:
            seen[:, list(gone)] = False
        k, v = B.rows(b)
        rows = [B.st[b] + i for i in at]
        check_rows(out[rows], *ref_rows(q[rows], k, v, seen), what=f"sequence {b}")


@pytest.mark.parametrize("H,rows,ps", [(80, 20, 16), (80, 20, 64), (64, 40, 32), (128, 32, 16)])   # 200, 320 and 512 rows
@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_ragged_batches(H, rows, ps, tree):
    """Batches cut into pieces of equal length: sequences of very different lengths, some without tokens or hardly any keys, a page
    that the pool does not have, NaN behind the sequences; then the same launch over other lengths, captured and replayed."""
    rng = random.Random(H + ps)
    news = [rows, 3, 0, rows - 1] + [rng.randrange(1, rows + 1) for _ in range(12)]
    lens = [4000, 3, 700, rows - 1, 64, 65, 128 + rows, 1500] + [rng.randrange(rows, 900) for _ in range(8)]
    news[4], news[5] = min(news[4], 64), min(news[5], 65)
    B = Batch(34, news, lens, ps, 8)
    used = torch.zeros(B.n_pages, ps, dtype=torch.bool, device="cuda")
    for b, L in enumerate(lens):
        at = torch.arange(L, device="cuda")
        used[B.t[b][at // ps].long(), at % ps] = True
    B.kp[~used], B.vp[~used] = float("nan"), float("inf")
    table = [list(r) for r in B.table]
    table[7][2] = B.n_pages + 5
    gone = list(range(2 * ps, 3 * ps))
    t = ints(table)
    T = sum(news)
    q = rnd(B.g, T, H, 128)
    trees = [random_tree(rng, n) for n in news]
    words = tree_words(trees, 1) if tree else None
    kw = dict(max_rows=rows, max_keys=16000, tree=words)
    need = cache.attention_ws_bytes(16, T, rows, B.width * ps, H, 8, ps)
    need = max(need, cache.attention_ws_bytes(16, T, rows, 16000, H, 8, ps))
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    wide = torch.cat([t, torch.full((16, 16000 // ps - B.width), -1, dtype=torch.int32, device="cuda")], 1)
    out = torch.full((T + 2, H, 128), 9.0, dtype=BF16, device="cuda")
    lens_t = B.lens.clone()
    call = lambda: cache.attention(q, B.kp, B.vp, wide, B.starts, lens_t, out[:T], workspace=ws, **kw)

    def check(L):
        for b, n in enumerate(news):
            if not n:
                continue
            at = sorted({0, n // 2, n - 1}) if L[b] > 300 else list(range(n))
            seen = (tree_seen(trees[b], L[b]) if tree else chain_seen(n, L[b]))[at]
            if b == 7:
                seen[:, [j for j in gone if j < L[b]]] = False
            p = torch.arange(L[b], device="cuda")
            page = B.t[b][p // ps].long()
            r = [B.st[b] + i for i in at]
            check_rows(out[r], *ref_rows(q[r], B.kp[page, p % ps], B.vp[page, p % ps], seen), what=f"sequence {b}")
        assert (out[T:] == 9.0).all() and (ws[need:] == 255).all()

    call()
    check(lens)
    first = out.clone()
    call()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    other = [max(n, L // 3) for n, L in zip(news, lens)]
    other[0] = 4000 if tree else rows      # (the longest stays, or is the first tokens alone)
    for L in (other, lens):
        lens_t.copy_(ints(L))
        out[:T].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check(L)
    assert torch.equal(out, first)


def test_a_tree_of_one_branch_is_a_chain():
    news, lens = [9, 70], [100, 70]
    B = Batch(13, news, lens, 16, 2)
    q = rnd(B.g, sum(news), 4, 128)
    trees = [[set(range(i + 1)) for i in range(n)] for n in news]
    a = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, tree=tree_words(trees, 2))
    B.check(q, a, lambda b: chain_seen(news[b], lens[b]))


@pads
@pytest.mark.parametrize("heads", [2, 40])
def test_masks_that_leave_a_row_empty(heads, pad):
    """A token whose mask has no bit, first with nothing before it (zeros), then behind a context."""
    B = Batch(14, [3, 3], [3, 40], 16, 1, pad=pad)
    q = rnd(B.g, 6, heads, 128)
    trees = [[{0}, set(), {0, 2}], [set(), {1}, {1, 2}]]
    out = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, tree=tree_words(trees, 1))
    assert (out[1] == 0).all()
    B.check(q, out, lambda b: tree_seen(trees[b], B.L[b]))


@pads
@pytest.mark.parametrize("news,lens,tree", [([1, 1], [70, 3000], False), ([6, 20], [70, 333], True), ([90], [200], False),
                                            ([6, 60], [70, 333], True)])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_positions_that_are_not_seen_have_no_part(news, lens, tree, what, pad):
    """Pages' rows behind the sequences' ends, free pages, and drafted tokens of other branches hold NaN or infinities."""
    B = Batch(15, news, lens, 16, 2, pad=pad)
    used = torch.zeros(B.n_pages, 16, dtype=torch.bool, device="cuda")
    for b, L in enumerate(lens):
        at = torch.arange(L, device="cuda")
        used[B.t[b][at // 16].long(), at % 16] = True
    B.kp[~used] = what
    B.vp[~used] = what
    rng = random.Random(6)
    trees = [random_tree(rng, n) for n in news]
    if tree:   # a leaf that no one but itself sees
        at = lens[1] - 1
        B.kp[B.table[1][at // 16], at % 16, 0] = what
        B.vp[B.table[1][at // 16], at % 16, 1] = what
    q = rnd(B.g, sum(news), 4, 128)
    kw = dict(tree=tree_words(trees, 1)) if tree else {}
    out = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, **kw)
    B.check(q, out, lambda b: tree_seen(trees[b], lens[b]) if tree else chain_seen(news[b], lens[b]))


@pads
@pytest.mark.parametrize("heads", [4, 80])
def test_pages_outside_the_pool_hold_nothing(heads, pad):
    """Entries below and past the pool's pages: their positions are not seen; a sequence of nothing else gets zeros."""
    news, lens = [1, 2, 1], [100, 60, 40]
    for ps in (16, 64, 8):
        B = Batch(16, news, lens, ps, 2, pad=pad)
        table = [list(r) for r in B.table]
        gone = [set(), set(), set()]
        for b, e, value in ((0, 1, -1), (0, 0, B.n_pages), (1, 0, 1 << 30), (2, None, -7)):
            for x in range(len(table[b])) if e is None else [min(e, -(-lens[b] // ps) - 1)]:
                table[b][x] = value
                gone[b] |= set(range(x * ps, (x + 1) * ps))
        q = rnd(B.g, 4, heads, 128)
        out = cache.attention(q, B.kp, B.vp, ints(table), B.starts, B.lens)

        def seen(b):
            s = chain_seen(news[b], lens[b])
            s[:, [j for j in gone[b] if j < lens[b]]] = False
            return s
        B.check(q, out, seen)
        assert (out[3] == 0).all()


@pads
@pytest.mark.parametrize("H", [4, 40])
def test_rows_behind_the_last_sequence_stay(H, pad):
    """A padded batch: more rows than tokens, a table wider than the sequences, sequences longer than the launch was sized
    for."""
    news, lens = [2, 1], [50, 3000]
    B = Batch(17, news, lens, 16, 1, pad=pad)
    q = rnd(B.g, 7, H, 128)
    out = torch.full((9, H, 128), 3.0, dtype=BF16, device="cuda")
    cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, out, max_rows=2)
    B.check(q, out, lambda b: chain_seen(news[b], lens[b]))
    assert (out[3:] == 3.0).all()
    # one token of the first sequence is beyond max_rows: its row stays as it was
    out.fill_(3.0)
    cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, out, max_rows=1)
    assert (out[1] == 3.0).all() and (out[3:] == 3.0).all() and not (out[0] == 3.0).any() and not (out[2] == 3.0).any()
    # positions beyond max_keys are not seen
    short = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, max_rows=2, max_keys=1000)
    k, v = B.rows(1)
    check_rows(short[2:3], *ref_rows(q[2:3], k[:1000], v[:1000], torch.ones(1, 1000, dtype=torch.bool)))
    # a length that the table does not hold
    lens2 = B.lens.clone()
    lens2[0] = 100000
    cut = cache.attention(q, B.kp, B.vp, B.t[:, :4].contiguous(), B.starts, lens2, max_rows=2)
    at = torch.arange(64, device="cuda")
    tab = B.t[0][at // 16].long()
    ok = tab >= 0
    k, v = B.kp[tab.clamp(min=0), at % 16], B.vp[tab.clamp(min=0), at % 16]
    check_rows(cut[:2], *ref_rows(q[:2], k, v, ok.cpu()[None].expand(2, 64)))


@pads
@pytest.mark.parametrize("ps", [16, 64])
def test_offsets_past_32_bits(ps, pad):
    """A pool of more than 2^31 elements whose last pages are the ones in use."""
    HK = 8
    pages = (1 << 31) // (ps * HK * 128) + 200
    kp, vp = (torch.zeros(pages, ps, HK, 128, dtype=BF16, device="cuda") for _ in range(2))
    for news, lens in (([1, 2], [500, 130]), ([30, 21], [300, 200])):      # few and many rows of a kv head
        B = Batch(18, news, lens, ps, HK, pad=pad)
        shift = pages - B.n_pages
        kp[shift:], vp[shift:] = B.kp, B.vp
        t = torch.where(B.t >= 0, B.t + shift, B.t)
        T = sum(news)
        q = rnd(B.g, T, 32, 128)
        out = cache.attention(q, kp, vp, t, B.starts, B.lens)
        B.check(q, out, lambda b: chain_seen(news[b], lens[b]))
        k, v = rnd(B.g, T, HK, 128), rnd(B.g, T, HK, 128)
        cache.append(None, k, v, kp, vp, t, B.starts, B.lens, table_kind=ops.TABLE_NONE)
        cache.append(None, k, v, B.kp, B.vp, B.t, B.starts, B.lens, table_kind=ops.TABLE_NONE)
        assert torch.equal(kp[shift:], B.kp) and torch.equal(vp[shift:], B.vp) and not kp[:4].any()
    cache.copy_pages(kp, vp, ints([B.table[0][0] + shift]), ints([1]))
    assert torch.equal(kp[1], B.kp[B.table[0][0]]) and torch.equal(vp[1], B.vp[B.table[0][0]])
    cache.move_rows(kp, vp, t, ints([0, 1, 1]), ints([5]), ints([250]))
    (p, r), (p2, r2) = divmod(5, ps), divmod(250, ps)
    assert torch.equal(kp[B.table[0][p2] + shift, r2], B.kp[B.table[0][p], r])
    del kp, vp
    torch.cuda.empty_cache()


def test_nothing_to_do():
    B = Batch(25, [0, 0], [5, 40], 16, 2)
    q, k = rnd(B.g, 0, 4, 128), rnd(B.g, 0, 2, 128)
    assert cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens).shape == (0, 4, 128)
    assert cache.append(q, k, k, B.kp, B.vp, B.t, B.starts, B.lens, table_kind=ops.TABLE_NONE).shape == (0, 4, 128)
    # rows but no tokens: nothing is written
    q = rnd(B.g, 3, 4, 128)
    out = torch.full((3, 4, 128), 2.0, dtype=BF16, device="cuda")
    before = B.kp.clone()
    cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, out)
    cache.append(q, q[:, :2], q[:, 2:], B.kp, B.vp, B.t, B.starts, B.lens, out, table_kind=ops.TABLE_NONE)
    assert (out == 2.0).all() and torch.equal(B.kp, before)


@pads
@pytest.mark.parametrize("many", [False, True])
def test_starts_and_lengths_that_make_no_sense(many, pad):
    """Whatever the device's integers say, nothing outside the tensors is read or written: sequences whose numbers are out of
    order or too large do less, the others are as always."""
    news, lens = [2, 30 if many else 3, 2], [200, 150, 90]
    B = Batch(26, news, lens, 16, 2, pad=pad)
    T = sum(news)
    q = rnd(B.g, T, 8, 128)
    good = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens)
    low, top = -(1 << 31), (1 << 31) - 1
    for st, ln in (([0, 2, T + 1000, 1 << 30], lens), ([-5, 2, T - 2, T], lens), (B.st[:4], [-3, 150, (1 << 30) + 7]),
                   ([T, T, 0, 0], lens), (B.st[:4], [1, 2, 1 << 29]), ([0, 2, low, T], lens), ([low, 2, top, low], lens),
                   ([0, 2, top, T], [low, top, top]), ([1, low, 1, top], [0, 0, 0])):
        st, ln = st + [st[-1]] * pad, ln + [top] * pad
        out = torch.full((T + 4, 8, 128), 6.0, dtype=BF16, device="cuda")
        cache.attention(q, B.kp, B.vp, B.t, ints(st), ints(ln), out[2:2 + T])
        assert (out[:2] == 6.0).all() and (out[2 + T:] == 6.0).all()
        k = rnd(B.g, T, 2, 128)
        kp, vp = B.kp.clone(), B.vp.clone()
        cache.append(q, k, k, kp, vp, B.t, ints(st), ints(ln), out[2:2 + T], table_kind=ops.TABLE_NONE)
        cache.move_rows(kp, vp, B.t, ints(st), ints([7] * T), ints([11] * T), max_rows=5)
        assert (out[:2] == 6.0).all() and (out[2 + T:] == 6.0).all()
    assert torch.equal(good, cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens))


@pads
@pytest.mark.parametrize("rows", [2, 4, 7, 20])
def test_drafted_tokens_beyond_max_rows_are_left_out(rows, pad):
    """As rows and as keys, on either side of the choices between the kernels."""
    n, L = 70, 300
    B = Batch(27, [n], [L], 16, 2, pad=pad)
    q = rnd(B.g, n, 16, 128)
    full = [set(range(n)) if i % 2 else set(range(0, n, 3)) for i in range(n)]
    tree = tree_words([full], 2)
    for window, sinks in ((0, 0), (50, 5)):
        out = torch.full((n, 16, 128), 6.0, dtype=BF16, device="cuda")
        cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, out, max_rows=rows, tree=tree, window=window, sinks=sinks)
        assert (out[rows:] == 6.0).all()
        seen = tree_seen(full, L, window, sinks)[:rows]
        seen[:, L - n + rows:] = False
        k, v = B.rows(0)
        check_rows(out[:rows], *ref_rows(q[:rows], k, v, seen))


@pytest.mark.parametrize("shape,perm", [((30, 2, 16, 2, 128), 1), ((30, 16, 2, 2, 128), 2), ((30, 16, 2, 2, 128), 3)])
@pads
def test_keys_and_values_in_one_buffer(shape, perm, pad):
    """Pages whose keys and values interleave page by page, token by token or head by head."""
    B = Batch(28, [2, 33], [120, 150], 16, 2, pages=30, pad=pad)
    both = rnd(B.g, *shape)
    kp, vp = both.unbind(perm)
    assert kp.shape == B.kp.shape
    kp.copy_(B.kp)
    vp.copy_(B.vp)
    q, k, v = rnd(B.g, 35, 8, 128), rnd(B.g, 35, 2, 128), rnd(B.g, 35, 2, 128)
    for kk, vv in ((kp, vp), (B.kp, B.vp)):
        cache.append(None, k, v, kk, vv, B.t, B.starts, B.lens, table_kind=ops.TABLE_NONE)
        cache.copy_pages(kk, vv, ints([0]), ints([1]))
        cache.move_rows(kk, vv, B.t, ints([0, 1, 3]), ints([5, 9, 70]), ints([6, 70, 9]))
    assert torch.equal(kp, B.kp) and torch.equal(vp, B.vp)
    for few in (slice(0, 2), slice(0, 35)):
        n = few.stop
        args = (B.t, ints([0, 2] + [n] * (pad + 1)), B.lens)
        assert torch.equal(cache.attention(q[few], kp, vp, *args), cache.attention(q[few], B.kp, B.vp, *args))


def test_a_captured_step_of_all_calls():
    """Append, attention (split over the keys, and of many rows), a move and a page copy in two graphs with workspaces of their own, replayed in
    turn with eager work between; every replay against the eager calls on copies."""
    B = Batch(29, [1, 40], [3000, 90], 16, 8)
    T, H = 41, 32
    q, k, v = rnd(B.g, T, H, 128), rnd(B.g, T, 8, 128), rnd(B.g, T, 8, 128)
    one = (ints([0, 1]), B.lens[:1])
    pairs = ints([B.table[1][5]]), ints([[p for p in range(B.n_pages) if p not in sum(B.table, [])][0]])
    moves = ints([0, 2, 3]), ints([7, 2999, 3]), ints([2999, 7, 88])

    def step(kp, vp, out, ws):
        cache.append(None, k, v, kp, vp, B.t, B.starts, B.lens, table_kind=ops.TABLE_NONE)
        cache.attention(q[:1], kp, vp, B.t, *one, out[:1], max_rows=1, max_keys=3000, workspace=ws)
        cache.attention(q, kp, vp, B.t, B.starts, B.lens, out[1:], max_rows=40, workspace=ws)
        cache.move_rows(kp, vp, B.t, *moves, max_rows=2)
        cache.copy_pages(kp, vp, *pairs)

    need = max(cache.attention_ws_bytes(1, 1, 1, 3000, H, 8, 16),
               cache.attention_ws_bytes(2, T, 40, B.width * 16, H, 8, 16))
    assert need > 0
    graphs = []
    for _ in range(2):
        kp, vp, out = B.kp.clone(), B.vp.clone(), torch.zeros(T + 1, H, 128, dtype=BF16, device="cuda")
        ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(kp, vp, out, ws)
        graphs.append((g, kp, vp, out, ws))
    ek, ev, eo = B.kp.clone(), B.vp.clone(), torch.zeros(T + 1, H, 128, dtype=BF16, device="cuda")
    ews = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for i in range(4):
        for x in (q, k, v):
            x.copy_(rnd(B.g, *x.shape))
        step(ek, ev, eo, ews)
        for g, kp, vp, out, ws in graphs:
            g.replay()
            torch.cuda.synchronize()
            rnd(B.g, 1000, 1000).sum().item()
            assert torch.equal(out, eo) and torch.equal(kp, ek) and torch.equal(vp, ev), f"replay {i}"


def test_workspace_streams_and_graphs():
    news, lens = [1, 1], [4000, 2500]
    B = Batch(19, news, lens, 16, 2)
    q = rnd(B.g, 2, 8, 128)
    args = (q, B.kp, B.vp, B.t, B.starts, B.lens)
    kw = dict(max_rows=1, max_keys=4000)
    want = cache.attention(*args, **kw)
    need = cache.attention_ws_bytes(2, 2, 1, 4000, 8, 2, 16)
    assert need > 0
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(cache.attention(*args, workspace=ws, **kw), want) and (ws[need:] == 255).all()
    with pytest.raises(ValueError):
        cache.attention(*args, workspace=ws[:need - 256], **kw)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            a = cache.attention(*args, **kw)
        b = cache.attention(*args, **kw)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)
    # a captured step follows tokens, lengths and tables at its replay
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attention(*args, out, **kw)
    for i, new_lens in enumerate(([4000, 2500], [37, 2500], [1, 900])):
        q.copy_(rnd(gen(60 + i), 2, 8, 128))
        B.lens.copy_(ints(new_lens))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cache.attention(*args, **kw))
        B.L = new_lens
        B.check(q, out, lambda b: chain_seen(1, new_lens[b]))


@pytest.mark.parametrize("news,lens,H,HK,rows,keys", [
    ([1, 1], [3900, 700], 32, 8, None, 6000),       # a table of fewer positions than max_keys says
    ([8] * 8, [900] * 7 + [3900], 32, 8, 128, None),   # fewer tokens than max_rows says: none needed for as many as that
])
def test_workspaces_of_larger_numbers(news, lens, H, HK, rows, keys):
    """A workspace of attention_ws_bytes for a max_rows or max_keys that is more than the tokens or the table is taken, also where the
    call itself would be cut into more parts."""
    B = Batch(37, news, lens, 16, HK)
    T = sum(news)
    q = rnd(B.g, T, H, 128)
    most = B.width * 16
    need = cache.attention_ws_bytes(len(news), T, rows or T, keys or most, H, HK, 16)
    assert need < cache.attention_ws_bytes(len(news), T, min(rows or T, T), min(keys or most, most), H, HK, 16)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    out = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, max_rows=rows, max_keys=keys, workspace=ws[:need])
    B.check(q, out, lambda b: chain_seen(news[b], lens[b]))
    assert (ws[need:] == 255).all()
    if need:
        with pytest.raises(ValueError, match="contiguous bytes on the current device needed"):
            cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, max_rows=rows, max_keys=keys, workspace=ws[:need - 256])


def test_the_same_call_gives_the_same_bits():
    B = Batch(20, [3, 1, 40], [2000, 700, 900], 16, 2)
    q = rnd(B.g, 44, 8, 128)
    a = cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens)
    assert all(torch.equal(a, cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens)) for _ in range(3))


# ------------------------------------------------------------------------------------------------ append
def tables(kind, rows, rot, g):
    ang = torch.rand(rows, rot // 2, generator=g, device="cuda", dtype=torch.float64) * 6.3
    c, s = ang.cos(), ang.sin()
    if kind == ops.TABLE_COSSIN_F32:
        c, s = c.float(), s.float()
        return (c, s), torch.stack([c, -s, s, c], -1).double()
    m = torch.stack([c, -s, s, c], -1).to(BF16 if kind == ops.TABLE_MAT2_BF16 else torch.float32)
    return (m.reshape(rows, 2 * rot).contiguous(), None), m.double()


def ref_norm_rope(x, w, mat, rot, pairing, eps):
    """(y, size) in fp64: the value and the size of what it is a sum of; mat [T, rot / 2, 4] or None."""
    x = x.double()
    y = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    size = y.abs()
    if mat is not None:
        a_at = torch.arange(0, rot, 2) if pairing == ops.PAIR_INTERLEAVED else torch.arange(rot // 2)
        b_at = a_at + (1 if pairing == ops.PAIR_INTERLEAVED else rot // 2)
        f = mat[:, None]
        a, b = y[..., a_at].clone(), y[..., b_at].clone()
        y[..., a_at], y[..., b_at] = f[..., 0] * a + f[..., 1] * b, f[..., 2] * a + f[..., 3] * b
        size[..., a_at] = size[..., b_at] = a.abs() + b.abs()
    return y, size


def close_rope(got, y, size, what):
    # one rounding to bf16, and fp32 steps before it: the sum of 128 squares, the root and three products and sums, below
    # 2^-17 of the values that are added
    over = (got.double() - y).abs() > HALF * y.abs() + 2.0 ** -16 * size + 1e-30
    assert not over.any(), f"{what}: {int(over.sum())} values off"


APPENDS = [   # tokens, lengths, heads, kv heads, page size, table kind, pairing, rot, weights, by_head
    ([1], [1], 1, 1, 16, ops.TABLE_COSSIN_F32, ops.PAIR_INTERLEAVED, 128, True, False),
    ([1] * 32, [7 + 11 * i for i in range(32)], 32, 8, 16, ops.TABLE_COSSIN_F32, ops.PAIR_INTERLEAVED, 128, True, False),
    ([5, 0, 0, 77, 1], [9, 3, 0, 300, 65], 7, 1, 64, ops.TABLE_COSSIN_F32, ops.PAIR_SPLIT_HALF, 96, False, True),
    ([130, 3], [130, 4], 6, 3, 1, ops.TABLE_MAT2_BF16, ops.PAIR_SPLIT_HALF, 128, True, False),
    ([40], [45], 5, 5, 8, ops.TABLE_MAT2_F32, ops.PAIR_INTERLEAVED, 64, True, False),
    ([33, 2], [40, 90], 4, 2, 32, ops.TABLE_NONE, ops.PAIR_INTERLEAVED, 128, True, True),
    ([i % 4 for i in range(300)], [5 + i for i in range(300)], 2, 1, 16, ops.TABLE_COSSIN_F32, ops.PAIR_INTERLEAVED, 32, True,
     False),
]


@pytest.mark.parametrize("c", APPENDS, ids=lambda c: f"{len(c[0])}seq{sum(c[0])}h{c[2]}g{c[3]}p{c[4]}k{c[5]}r{c[7]}")
def test_append(c):
    news, lens, H, HK, ps, kind, pairing, rot, weights, by_head = c
    B = Batch(21, news, lens, ps, HK, by_head)
    T = sum(news)
    qkv = rnd(B.g, T, H + 2 * HK, 128)
    q, k, v = qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:]
    wq, wk = ((torch.rand(128, generator=B.g, device="cuda") + 0.5 for _ in range(2)) if weights else (None, None))
    table, mat = tables(kind, max(lens), rot, B.g) if kind else (None, None)
    tok_b = [b for b, n in enumerate(news) for _ in range(n)]
    slots = torch.tensor([lens[b] - n + i for b, n in enumerate(news) for i in range(n)], device="cuda")
    page = B.t[torch.tensor(tok_b, device="cuda"), slots // ps].long()
    want_k, want_v = B.kp.clone(), B.vp.clone()
    kw = dict(q_norm=wq, k_norm=wk, table_kind=kind, table=table, pairing=pairing, rot=rot, eps=1e-5)
    before_k, before_v = B.kp.clone(), B.vp.clone()
    q_out = cache.append(q, k, v, B.kp, B.vp, B.t, B.starts, B.lens, **kw)
    rows = mat[slots] if kind else None
    close_rope(q_out, *ref_norm_rope(q, wq, rows, rot, pairing, 1e-5), "queries")
    close_rope(B.kp[page, slots % ps], *ref_norm_rope(k, wk, rows, rot, pairing, 1e-5), "keys")
    assert torch.equal(B.vp[page, slots % ps], v)
    want_k[page, slots % ps], want_v[page, slots % ps] = B.kp[page, slots % ps], v
    assert torch.equal(B.kp, want_k) and torch.equal(B.vp, want_v)      # nothing else was written
    # keys and values alone, and the queries in place
    k2, v2 = before_k.clone(memory_format=torch.preserve_format), before_v.clone(memory_format=torch.preserve_format)
    assert cache.append(None, k, v, k2, v2, B.t, B.starts, B.lens, **kw) is None
    assert torch.equal(k2, B.kp) and torch.equal(v2, B.vp)
    keep = qkv[:, H:].clone()
    cache.append(q, k, v, B.kp, B.vp, B.t, B.starts, B.lens, q, **kw)
    assert torch.equal(q, q_out) and torch.equal(qkv[:, H:], keep) and torch.equal(B.kp, want_k)


def test_append_queries_are_joint_q_prepares():
    """The same arithmetic as the fused op's query launch, bit for bit."""
    B = Batch(22, [50], [50], 16, 2)
    q, k = rnd(B.g, 50, 4, 128), rnd(B.g, 50, 2, 128)
    w = torch.rand(128, generator=B.g, device="cuda")
    cos, sin = (torch.from_numpy(x).cuda() for x in rope.grid2d_table(10, 5, 8))
    a = cache.append(q, k, k, B.kp, B.vp, B.t, B.starts, B.lens, q_norm=w, k_norm=w, table=(cos, sin))
    assert torch.equal(a, ops.joint_q_prepare(q, q_norm=w, q_table=(cos, sin)))
    assert torch.equal(B.rows(0)[0], ops.joint_q_prepare(k, q_norm=w, q_table=(cos, sin)))


def test_append_leaves_out_what_has_no_place():
    """Tokens whose position, page or table row does not exist, and rows behind the last sequence."""
    news, lens = [3, 2, 2], [20, 18, 5]
    B = Batch(23, news, lens, 8, 1)
    table = [list(r) for r in B.table]
    table[0][2] = B.n_pages                      # positions 16 .. of sequence 0: tokens 17, 18, 19
    q, k = rnd(B.g, 9, 2, 128), rnd(B.g, 9, 1, 128)
    tab, _ = tables(ops.TABLE_COSSIN_F32, 17, 128, B.g)        # sequence 1's last token (position 17) has no row
    before_k, before_v = B.kp.clone(), B.vp.clone()
    out = torch.full((9, 2, 128), 4.0, dtype=BF16, device="cuda")
    cache.append(q, k, k, B.kp, B.vp, ints(table), B.starts, B.lens, out, table=tab)
    done = [(3, 1, 16), (5, 2, 3), (6, 2, 4)]    # token, sequence, position
    for t in range(9):
        assert (out[t] == 4.0).all() == (t not in [d[0] for d in done])
    for t, b, p in done:
        assert torch.equal(B.vp[table[b][p // 8], p % 8], k[t])
        before_k[table[b][p // 8], p % 8] = B.kp[table[b][p // 8], p % 8]
        before_v[table[b][p // 8], p % 8] = k[t]
    assert torch.equal(B.kp, before_k) and torch.equal(B.vp, before_v)
    # explicit positions choose the table row; those outside the table leave the token out
    pos = ints([0, 0, 0, 5, 16, 17, -1, 3, 3])
    out.fill_(4.0)
    cache.append(q, k, k, B.kp, B.vp, B.t, B.starts, B.lens, out, table=tab, positions=pos)
    assert (out[5:] == 4.0).all() and not (out[:5] == 4.0).all(-1).any()
    same = cache.append(q[3:5], k[3:5], k[3:5], B.kp, B.vp, B.t[2:], ints([0, 2]), B.lens[2:],
                        table=(tab[0][[5, 16]].contiguous(), tab[1][[5, 16]].contiguous()), positions=ints([0, 1]))
    assert torch.equal(out[3:5], same)


def test_append_in_place_needs_columns_of_its_own():
    B = Batch(36, [5, 4], [20, 11], 16, 2)
    qkv = rnd(B.g, 9, 8, 128)
    args = (B.kp, B.vp, B.t, B.starts, B.lens)
    for k, v in ((qkv[:, :2], qkv[:, 6:]), (qkv[:, 4:6], qkv[:, 3:5])):
        with pytest.raises(_lib.LrError):
            cache.append(qkv[:, :4], k, v, *args, qkv[:, :4], table_kind=ops.TABLE_NONE)
    want_k, want_v = B.kp.clone(), B.vp.clone()
    want = cache.append(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], want_k, want_v, *args[2:], table_kind=ops.TABLE_NONE)
    keep = qkv[:, 4:].clone()
    cache.append(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], *args, qkv[:, :4], table_kind=ops.TABLE_NONE)
    assert torch.equal(qkv[:, :4], want) and torch.equal(qkv[:, 4:], keep)
    assert torch.equal(B.kp, want_k) and torch.equal(B.vp, want_v)


def test_append_of_column_views_of_a_table():
    """cos and sin as columns of a wider table: the view's columns count, not its rows' stride. Too narrow ones are refused, and
    nothing is written."""
    B = Batch(35, [3], [20], 16, 1)
    q, k = rnd(B.g, 3, 2, 128), rnd(B.g, 3, 1, 128)
    (cos, sin), _ = tables(ops.TABLE_COSSIN_F32, 20, 128, B.g)
    wide = torch.cat([cos, sin, cos], 1)
    before_k, before_v = B.kp.clone(), B.vp.clone()
    for a, b in ((cos[:, 32:], sin[:, 32:]), (wide[:, 129:], wide[:, 129:]), (wide[:, :32], wide[:, 64:96])):
        with pytest.raises(ValueError, match="table: rows of"):
            cache.append(q, k, k, B.kp, B.vp, B.t, B.starts, B.lens, table=(a, b))
    assert torch.equal(B.kp, before_k) and torch.equal(B.vp, before_v)
    got = cache.append(q, k, k, B.kp, B.vp, B.t, B.starts, B.lens, table=(wide[:, :64], wide[:, 64:128]))
    keys = B.kp.clone()
    assert torch.equal(got, cache.append(q, k, k, B.kp, B.vp, B.t, B.starts, B.lens, table=(cos, sin))) and torch.equal(keys, B.kp)
    half = cache.append(q, k, k, B.kp, B.vp, B.t, B.starts, B.lens, table=(cos[:, 32:], sin[:, 32:]), rot=64)
    assert torch.equal(half, cache.append(q, k, k, B.kp, B.vp, B.t, B.starts, B.lens, rot=64,
                                          table=(cos[:, 32:].contiguous(), sin[:, 32:].contiguous())))


# ------------------------------------------------------------------------------------------------ copies and moves
@pytest.mark.parametrize("ps,HK,by_head,layers", [(16, 8, False, 3), (1, 1, False, None), (64, 3, True, 2), (128, 5, False, 1),
                                                  (8, 7, True, None)])
def test_copy_pages(ps, HK, by_head, layers):
    g = gen(30)
    kp, vp = make_pool(g, 12, ps, HK, by_head, layers)
    src, dst = [3, 3, 0, 11, -1, 5, 12, 7], [1, 2, 9, 4, 6, 12, 8, 7]
    wk, wv = kp.clone(), vp.clone()
    for a, b in zip(src, dst):
        if 0 <= a < 12 and 0 <= b < 12:
            wk[..., b, :, :, :], wv[..., b, :, :, :] = kp[..., a, :, :, :], vp[..., a, :, :, :]
    cache.copy_pages(kp, vp, ints(src), ints(dst))
    assert torch.equal(kp, wk) and torch.equal(vp, wv)
    cache.copy_pages(kp, vp, ints([]), ints([]))
    with pytest.raises(ValueError):
        cache.copy_pages(kp, vp, ints([1]), ints([1, 2]))


@pytest.mark.parametrize("ps,HK,by_head,layers,counts", [
    (16, 8, False, 3, [5, 0, 1]), (1, 2, False, 1, [30, 2, 7]), (64, 3, True, 2, [256, 1, 9]), (8, 40, False, None, [100, 3, 3])])
def test_move_rows(ps, HK, by_head, layers, counts):
    """Chains, swaps and gathers inside sequences: every row is read before any is written."""
    lens = [300, 40, 90]
    g, rng = gen(31), random.Random(8)
    need = [-(-x // ps) for x in lens]
    ids = list(range(sum(need) + 2))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(n)] + [-1] * (max(need) - n) for n in need]
    kp, vp = make_pool(g, sum(need) + 2, ps, HK, by_head, layers)
    src, dst, st = [], [], [0]
    for L, n in zip(lens, counts):
        to = rng.sample(range(L), n)                       # distinct targets, sources as they come: chains, swaps, repeats
        src += [rng.choice(to) if rng.random() < 0.5 else rng.randrange(L) for _ in range(n)]
        dst += to
        st.append(st[-1] + n)
    if counts[2] >= 3:                                     # places that do not exist: left out
        src[-1], dst[-2], src[-3] = -1, lens[2] + 1000, 1 << 30
    wk, wv = kp.clone(), vp.clone()
    for b in range(3):
        for a, c in zip(src[st[b]:st[b + 1]], dst[st[b]:st[b + 1]]):
            if 0 <= a < lens[b] and 0 <= c < lens[b]:
                (pa, ra), (pc, rc) = divmod(a, ps), divmod(c, ps)
                wk[..., table[b][pc], rc, :, :] = kp[..., table[b][pa], ra, :, :]
                wv[..., table[b][pc], rc, :, :] = vp[..., table[b][pa], ra, :, :]
    cache.move_rows(kp, vp, ints(table), ints(st), ints(src), ints(dst), max_rows=max(counts))
    assert torch.equal(kp, wk) and torch.equal(vp, wv)


def test_refusals_before_launch():
    B = Batch(32, [1], [20], 16, 2)
    q = rnd(B.g, 1, 4, 128)
    ok = (q, B.kp, B.vp, B.t, B.starts, B.lens)
    with pytest.raises(_lib.LrError):
        cache.attention(*ok, q)                                        # in place
    with pytest.raises(_lib.LrError):
        cache.attention(*ok, scale=-1.0)
    with pytest.raises(ValueError):
        cache.attention(q, B.kp, B.vp[:1], *ok[3:])
    with pytest.raises(ValueError):
        cache.attention(q, B.kp, B.vp.transpose(1, 2).contiguous().transpose(1, 2), *ok[3:])   # other strides
    with pytest.raises(ValueError):
        cache.attention(q, B.kp.float(), B.vp.float(), *ok[3:])
    with pytest.raises(ValueError):
        cache.attention(q, B.kp, B.vp, B.t.long(), B.starts, B.lens)
    with pytest.raises(ValueError):
        cache.attention(q, B.kp, B.vp, B.t, B.starts.cpu(), B.lens)
    with pytest.raises(ValueError):
        cache.attention(*ok, tree=torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(_lib.LrError):
        cache.append(q[:, :2], B.kp[0, :1], B.vp[0, :1], *ok[1:], table_kind=ops.TABLE_NONE)    # k inside the pool
    with pytest.raises(ValueError):
        cache.append(q, q, q, *ok[1:], table_kind=ops.TABLE_NONE)      # four key heads over a pool of two
    odd = rnd(B.g, 3, 12, 2, 128)
    with pytest.raises(_lib.LrError):
        cache.attention(q, odd, odd.clone(), *ok[3:])                  # pages of 12 rows
    with pytest.raises(_lib.LrError):
        cache.move_rows(B.kp, B.vp, B.t, ints([0, 300]), ints([0] * 300), ints([0] * 300))


def test_numbers_past_32_bits_are_refused():
    B = Batch(33, [1], [20], 16, 2)
    q = rnd(B.g, 1, 4, 128)
    for kw in (dict(window=1 << 32), dict(window=4, sinks=(1 << 32) + 4)):
        with pytest.raises(ValueError):
            cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, **kw)
    for kw in (dict(max_rows=5 - (1 << 33)), dict(max_keys=-(1 << 40) + 20), dict(max_rows=0), dict(max_keys=-1)):
        with pytest.raises(_lib.LrError):
            cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, **kw)
    assert torch.equal(cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens, max_rows=1 << 40, max_keys=1 << 40),
                       cache.attention(q, B.kp, B.vp, B.t, B.starts, B.lens))
    for kw in (dict(window=1 << 32), dict(window=4, sinks=1 << 31), dict(window=4, frame=(1 << 32) + 1),
               dict(window=4, p0=1 << 32)):
        with pytest.raises(ValueError):
            ops.attention_window(q, B.kp[0], B.vp[0], **kw)


# ------------------------------------------------------------------------------------------------ together
def test_a_serving_loop():
    """Two layers of one model: prompts appended and attended, one request forked (its shared last page copied), drafted trees
    appended, attended and the accepted branch moved behind the context, then single tokens, in a window of 60 at the end;
    every attention against rows kept aside."""
    L, H, HK, ps, window, sinks = 2, 4, 2, 8, 60, 3
    g, rng = gen(40), random.Random(9)
    pool = cache.PagePool(64)
    kp, vp = make_pool(g, 64, ps, HK, layers=L)
    (cos, sin), _ = tables(ops.TABLE_COSSIN_F32, 256, 128, g)
    w = torch.rand(128, generator=g, device="cuda") + 0.5
    keys = [[] for _ in range(L)]                     # per layer, per sequence: (k, v) rows as written
    pages, lens = [], []

    def grow(b, n):
        while len(pages[b]) * ps < lens[b] + n:
            pages[b] += pool.alloc(1)
        lens[b] += n

    def args():
        width = max(map(len, pages))
        return ints([p + [-1] * (width - len(p)) for p in pages])

    def step(news, trees=None, window=0):
        """One forward of news[b] tokens each: append and attention in every layer, checked."""
        for b, n in enumerate(news):
            grow(b, n)
        st = [0]
        for n in news:
            st.append(st[-1] + n)
        t, starts, ln = args(), ints(st), ints(lens)
        ctx = [x - n for x, n in zip(lens, news)]
        depth = [ctx[b] + (len(trees[b][i]) - 1 if trees else i) for b, n in enumerate(news) for i in range(n)]
        for layer in range(L):
            qkv = rnd(g, st[-1], H + 2 * HK, 128)
            q = cache.append(qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:], kp[layer], vp[layer], t, starts, ln, q_norm=w,
                             k_norm=w, table=(cos, sin), positions=ints(depth))
            kk = ops.joint_q_prepare(qkv[:, H:H + HK], q_norm=w, q_table=(cos[depth].contiguous(), sin[depth].contiguous()))
            out = cache.attention(q, kp[layer], vp[layer], t, starts, ln, max_rows=max(news), max_keys=max(lens),
                                  tree=tree_words(trees, 1) if trees else None, window=window, sinks=sinks if window else 0)
            for b, n in enumerate(news):
                s = slice(st[b], st[b + 1])
                old = keys[layer][b] if b < len(keys[layer]) else (kk[:0], kk[:0])
                k2, v2 = torch.cat([old[0], kk[s]]), torch.cat([old[1], qkv[s, H + HK:]])
                seen = tree_seen(trees[b], lens[b], window, sinks) if trees else chain_seen(n, lens[b], window, sinks)
                check_rows(out[s], *ref_rows(q[s], k2, v2, seen), what=f"layer {layer} sequence {b}")
                if b < len(keys[layer]):
                    keys[layer][b] = (k2, v2)
                else:
                    keys[layer].append((k2, v2))

    pages += [[], []]
    lens += [0, 0]
    step([37, 70])
    # fork the first request: shared pages, its partly filled last page copied for the new one
    pages.append(pool.fork(pages[0]))
    lens.append(lens[0])
    src, dst = pool.own(pages[2], len(pages[2]) - 1)
    cache.copy_pages(kp, vp, ints([src]), ints([dst]))
    for layer in range(L):
        keys[layer].append(keys[layer][0])
    step([1, 1, 1])
    for _ in range(2):
        trees = [random_tree(rng, n) for n in (9, 14, 5)]
        before = list(lens)
        step([9, 14, 5], trees)
        paths = [sorted(rng.choice(t)) for t in trees]      # an accepted branch: a token's ancestors and itself
        moves = [(before[b] + x, before[b] + i) for b, p in enumerate(paths) for i, x in enumerate(p)]
        st = [0]
        for p in paths:
            st.append(st[-1] + len(p))
        cache.move_rows(kp, vp, args(), ints(st), ints([m[0] for m in moves]), ints([m[1] for m in moves]))
        for b, p in enumerate(paths):
            lens[b] = before[b] + len(p)
            at = torch.tensor(list(range(before[b])) + [before[b] + x for x in p], device="cuda")
            for layer in range(L):
                keys[layer][b] = tuple(x[at] for x in keys[layer][b])
            drop = len(pages[b]) - -(-lens[b] // ps)         # pages behind the accepted tokens
            if drop:
                pool.free(pages[b][-drop:])
                del pages[b][-drop:]
        step([1, 1, 1])
    # the second request ends; the pool is compacted
    pool.free(pages[1])
    gone = 1
    del pages[gone], lens[gone]
    for layer in range(L):
        del keys[layer][gone]
    a, b = pool.compact(pages)
    assert a
    cache.copy_pages(kp, vp, ints(a), ints(b))
    step([1, 1], window=window)
    step([3, 2], window=window)
