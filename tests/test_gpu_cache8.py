"""The cache in 8-bit pages on the GPU: appends against a 64-bit restatement of the format, attention against a 64-bit attention over
exactly what the pages hold, copies, and a serving loop of them together."""
from __future__ import annotations

import random

import pytest
import torch

from localrouter_amd import _lib, cache, ops
from tests.cache8_util import E8, F8, GROUP, exponent, exps, pack, scales_of, to_f8, values
from tests.cache_util import check_rows, gen, ref_rows, rnd
from tests.test_gpu_cache import Batch, chain_seen, ints, pads, random_tree, tree_seen, tree_words

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


class Batch8(Batch):
    """Sequences over a pool in 8 bits: the parent's pools, heads of different magnitude, packed."""

    def __init__(self, seed, news, lens, ps, HK, by_head=False, **kw):
        super().__init__(seed, news, lens, ps, HK, by_head, **kw)
        mag = torch.exp2(torch.arange(HK, device="cuda") % 5 - 2.0)[:, None]
        (self.kp, self.ks), (self.vp, self.vs) = (self._packed(p * m, by_head) for p, m in ((self.kp, 1.0), (self.vp, mag)))

    @staticmethod
    def _packed(p, by_head):
        q, s = pack(p.to(BF16))
        return (q.transpose(1, 2).contiguous().transpose(1, 2) if by_head else q.contiguous()), s.contiguous()

    def rows(self, b):
        at = torch.arange(self.L[b], device="cuda")
        page, row = self.t[b][at // self.ps].long().clamp(0, self.n_pages - 1), at % self.ps
        return values(self.kp, self.ks)[page, row], values(self.vp, self.vs)[page, row]

    def attend(self, q, **kw):
        return cache.attention_f8(q, self.kp, self.vp, self.ks, self.vs, kw.pop("table", self.t), self.starts, self.lens, **kw)


# ------------------------------------------------------------------------------------------------ attention
# tokens of each sequence, lengths, heads, kv heads, page size, window, sinks, by_head
CHAINS = [
    ([1], [1], 1, 1, 16, 0, 0, False),
    ([1], [16], 2, 1, 16, 0, 0, False),
    ([1], [17], 4, 1, 32, 0, 0, False),
    ([1], [777], 8, 2, 16, 0, 0, False),
    ([1], [5000], 4, 4, 64, 0, 0, False),                                   # split over the keys
    ([1, 1, 1], [33, 1, 400], 7, 1, 16, 0, 0, True),
    ([1, 0, 1, 1], [64, 5, 100, 31], 8, 8, 32, 0, 0, False),                # a sequence without tokens
    ([3, 1, 7], [3, 90, 7], 4, 2, 16, 0, 0, False),                         # prompts without context
    ([20, 33, 1], [220, 33, 65], 6, 2, 16, 0, 0, False),
    ([150, 9], [150, 300], 4, 1, 128, 0, 0, True),
    ([1, 1], [900, 2000], 8, 2, 16, 100, 4, False),
    ([40, 17], [300, 170], 4, 2, 32, 33, 7, False),
    ([5], [4000], 16, 1, 256, 1500, 1, True),
    ([1] * 40, [50 + 13 * i for i in range(40)], 2, 1, 16, 0, 0, False),
    ([2], [3000], 64, 1, 16, 0, 0, False),                                  # 128 rows of one kv head
    ([700, 333], [700, 1500], 4, 2, 16, 0, 0, False),                       # a prompt, and a chunk behind a context
    ([300], [1300], 8, 8, 64, 0, 0, True),
]


@pads
@pytest.mark.parametrize("c", CHAINS, ids=lambda c: f"{len(c[0])}seq{max(c[0])}of{max(c[1])}h{c[2]}g{c[3]}p{c[4]}w{c[5]}")
def test_attention_of_chains(c, pad):
    news, lens, H, HK, ps, window, sinks, by_head = c
    B = Batch8(11, news, lens, ps, HK, by_head, pad=pad)
    q = rnd(B.g, sum(news), H, 128)
    out = B.attend(q, max_rows=max(news), max_keys=max(lens), window=window, sinks=sinks)
    B.check(q, out, lambda b: chain_seen(news[b], lens[b], window, sinks))
    # nothing but the tensors: the table's own limits size the launch
    loose = B.attend(q, window=window, sinks=sinks)
    B.check(q, loose, lambda b: chain_seen(news[b], lens[b], window, sinks))


TREES = [
    ([5], [5], 4, 2, 16, 0, 0),             # a tree and nothing before it
    ([26, 11, 1], [300, 47, 200], 8, 2, 16, 0, 0),
    ([64], [1000], 8, 1, 32, 0, 0),
    ([65, 30], [165, 63], 2, 1, 16, 0, 0),  # two words
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
    B = Batch8(12, news, lens, ps, HK, pad=pad)
    q = rnd(B.g, sum(news), H, 128)
    out = B.attend(q, max_rows=max(news), tree=tree_words(trees, (max(news) + 63) // 64), window=window, sinks=sinks)
    B.check(q, out, lambda b: tree_seen(trees[b], lens[b], window, sinks))


@pytest.mark.parametrize("ps", [16, 64])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_many_rows(ps, tree):
    """8 sequences of 64 tokens x 128 heads over 8: the first and last tokens of some checked, with a page that the pool does not
    have."""
    news, lens = [64, 40, 64, 1, 64, 64, 50, 64], [4300, 5000, 64, 4100, 4200, 130, 4999, 2500]
    B = Batch8(24, news, lens, ps, 8)
    rng = random.Random(7)
    trees = [random_tree(rng, n) for n in news]
    table = [list(r) for r in B.table]
    table[6][3] = -5
    gone = range(3 * ps, 4 * ps)
    q = rnd(B.g, sum(news), 128, 128)
    out = B.attend(q, table=ints(table), max_rows=64, max_keys=5000, tree=tree_words(trees, 1) if tree else None)
    for b in (0, 2, 3, 6):
        at = sorted({0, min(1, news[b] - 1), news[b] - 1})
        seen = (tree_seen(trees[b], lens[b]) if tree else chain_seen(news[b], lens[b]))[at]
        if b == 6:
            seen[:, list(gone)] = False
        k, v = B.rows(b)
        rows = [B.st[b] + i for i in at]
        check_rows(out[rows], *ref_rows(q[rows], k, v, seen), what=f"sequence {b}")


BLOCK_SHARES = [
    # heads, kv heads, tokens, lengths, page, tree, of sizes for
    (128, 8, [290], [4500], 16, False, (290, 4500)),
    (128, 8, [600], [5555], 32, False, (600, 5555)),          # more blocks than an XCD has places
    (64, 8, [320, 300], [5700, 5200], 16, False, (320, 5700)),
    (56, 8, [320, 0], [4999, 70], 64, False, (350, 9000)),    # a sequence without tokens, fewer positions than the call is sized for
    (56, 8, [3, 345], [3, 700], 64, False, (350, 9000)),      # short shares: several of them, and the end of the row of blocks, empty
    (72, 4, [277, 241], [277, 4100], 128, False, (280, 4100)),   # a prompt without context
    (64, 8, [300, 320], [4700, 400], 16, True, (320, 4800)),
    (64, 8, [205, 1, 190], [5100, 4000, 190], 32, True, (205, 5100)),
]


@pytest.mark.parametrize("c", BLOCK_SHARES, ids=lambda c: f"{len(c[2])}seq{max(c[2])}of{max(c[3])}h{c[0]}g{c[1]}p{c[4]}t{int(c[5])}")
def test_attention_of_chunks_in_equal_shares(c):
    """Blocks of rows that do not fill the chip's places evenly, cut into equal shares of their tiles: some tokens of each sequence
    checked, a page that the pool does not have, NaN behind the sequences; bit for bit again, and as rows of a captured call over other
    lengths."""
    H, HK, news, lens, ps, tree, (rows, most) = c
    rng = random.Random(H)
    X = Batch8(26, news, lens, ps, HK)
    used = torch.zeros(X.n_pages, ps, dtype=torch.bool, device="cuda")
    for b, L in enumerate(lens):
        at = torch.arange(L, device="cuda")
        used[X.t[b][at // ps].long(), at % ps] = True
    X.kp.view(torch.uint8)[~used], X.vp.view(torch.uint8)[~used] = 0x7f, 0xff
    table = torch.full((len(news), max(X.width, -(-most // ps))), -1, dtype=torch.int32, device="cuda")
    table[:, :X.width] = X.t
    gone = list(range(ps, 2 * ps)) if lens[0] > 2 * ps else []
    if gone:
        table[0, 1] = X.n_pages + 5
    T = sum(news)
    q = rnd(X.g, T, H, 128)
    trees = [random_tree(rng, n) for n in news]
    kw = dict(max_rows=rows, max_keys=most, tree=tree_words(trees, (rows + 63) // 64) if tree else None)
    need = cache.attention_f8_ws_bytes(len(news), T, rows, most, H, HK, ps)
    assert need
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((T + 2, H, 128), 9.0, dtype=BF16, device="cuda")
    lens_t = X.lens.clone()
    call = lambda: cache.attention_f8(q, X.kp, X.vp, X.ks, X.vs, table, X.starts, lens_t, out[:T], workspace=ws, **kw)

    def check(L):
        k8, v8 = values(X.kp, X.ks), values(X.vp, X.vs)
        for b, n in enumerate(news):
            if not n:
                continue
            at = sorted({0, n // 3, n // 2, n - 1})
            seen = (tree_seen(trees[b], L[b]) if tree else chain_seen(n, L[b]))[at]
            if b == 0:
                seen[:, [j for j in gone if j < L[b]]] = False
            p = torch.arange(L[b], device="cuda")
            page = X.t[b][p // ps].long()
            r = [X.st[b] + i for i in at]
            check_rows(out[r], *ref_rows(q[r], k8[page, p % ps], v8[page, p % ps], seen), what=f"sequence {b}")
        assert (out[T:] == 9.0).all() and (ws[need:] == 255).all() and out.isfinite().all()

    call()
    check(lens)
    first = out.clone()
    out[:T].fill_(7.0)
    call()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for L in ([max(n, x // 3) for n, x in zip(news, lens)], lens):
        lens_t.copy_(ints(L))
        out[:T].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check(L)
    assert torch.equal(out, first)


CHUNKS = [
    # tokens of each sequence, lengths, heads, kv heads, page size, window, sinks, by_head, tree: more than 600 blocks of 32 rows
    ([700, 333], [700, 1500], 32, 2, 16, 0, 0, False, False),
    ([300], [1300], 128, 4, 64, 0, 0, True, False),
    ([400, 170], [3000, 170], 64, 4, 32, 333, 7, False, False),
    ([256, 200, 1, 0, 256, 30, 256, 99], [8000, 4000, 900, 50, 5000, 30, 256, 6500], 32, 8, 64, 0, 0, False, False),
    ([250], [2600], 96, 3, 128, 1000, 4, True, False),
    ([180, 220], [900, 4000], 64, 2, 16, 0, 0, False, True),
    ([220], [1700], 100, 4, 256, 600, 5, False, True),
    ([900], [900], 40, 1, 16, 0, 0, False, False),
]


@pads
@pytest.mark.parametrize("c", CHUNKS, ids=lambda c: f"{len(c[0])}seq{max(c[0])}of{max(c[1])}h{c[2]}g{c[3]}p{c[4]}w{c[5]}t{int(c[8])}")
def test_attention_of_chunks(c, pad):
    news, lens, H, HK, ps, window, sinks, by_head, tree = c
    B = Batch8(31, news, lens, ps, HK, by_head, pad=pad)
    rng = random.Random(8)
    trees = [random_tree(rng, n) for n in news]
    q = rnd(B.g, sum(news), H, 128)
    out = B.attend(q, max_rows=max(news), max_keys=max(lens), tree=tree_words(trees, (max(news) + 63) // 64) if tree else None, window=window,
                   sinks=sinks)
    for b, n in enumerate(news):
        at = sorted({i for i in (0, 1, n // 3, n // 2, n - 1) if 0 <= i < n})
        if not at:
            continue
        seen = (tree_seen(trees[b], lens[b], window, sinks) if tree else chain_seen(n, lens[b], window, sinks))[at]
        k, v = B.rows(b)
        rows = [B.st[b] + i for i in at]
        check_rows(out[rows], *ref_rows(q[rows], k, v, seen), what=f"sequence {b}")


SHARES = [
    # heads, kv heads, tokens, page, window, sinks, tree, long sequences
    (32, 8, 1, 16, 0, 0, False, 2),
    (32, 8, 1, 64, 700, 5, False, 3),
    (8, 8, 2, 32, 0, 0, False, 1),
    (16, 4, 4, 16, 0, 0, True, 2),
    (24, 8, 9, 32, 0, 0, True, 2),          # 27 rows of a kv head
    (24, 8, 9, 16, 300, 4, True, 2),
    (64, 8, 4, 16, 0, 0, False, 2),         # 32
    (4, 1, 3, 16, 0, 0, False, 4),          # an odd number of kv heads
    (21, 7, 5, 32, 0, 0, False, 1),
    (35, 7, 5, 32, 0, 0, True, 3),          # 25 rows
]


@pytest.mark.parametrize("c", SHARES, ids=lambda c: f"h{c[0]}g{c[1]}n{c[2]}p{c[3]}w{c[4]}t{int(c[6])}l{c[7]}")
@pytest.mark.parametrize("B", [16, 64])
def test_attention_of_batches_in_equal_shares(c, B):
    """Batches sized for long sequences: shares that hold many short pairs, pairs of many shares, sequences without tokens, a page that
    the pool does not have, NaN behind the sequences; then the same launch over other lengths, captured and replayed; bit for bit again
    in the same workspace."""
    H, HK, rows, ps, window, sinks, tree, longs = c
    rng = random.Random(H + B)
    news = [rows] + [rng.randrange(0, rows + 1) for _ in range(B - 1)]
    lens = [3000 + 97 * i for i in range(longs)] + [rng.randrange(rows, 70) for _ in range(B - longs)]
    news[longs - 1], lens[-1], news[-1] = rows, rows, rows
    X = Batch8(25, news, lens, ps, HK)
    used = torch.zeros(X.n_pages, ps, dtype=torch.bool, device="cuda")
    for b, L in enumerate(lens):
        at = torch.arange(L, device="cuda")
        used[X.t[b][at // ps].long(), at % ps] = True
    X.kp.view(torch.uint8)[~used], X.vp.view(torch.uint8)[~used] = 0x7f, 0xff
    most = 32 * -(-32768 // (B * HK))
    table = torch.full((B, max(X.width, -(-most // ps))), -1, dtype=torch.int32, device="cuda")
    table[:, :X.width] = X.t
    gone = list(range(2 * ps, 3 * ps)) if longs > 1 else []
    if gone:
        table[0, 2] = X.n_pages + 5
    T = sum(news)
    q = rnd(X.g, T, H, 128)
    trees = [random_tree(rng, n) for n in news]
    kw = dict(max_rows=rows, max_keys=max(most, max(lens)), tree=tree_words(trees, 1) if tree else None, window=window, sinks=sinks)
    need = cache.attention_f8_ws_bytes(B, T, rows, kw["max_keys"], H, HK, ps, window=window, sinks=sinks)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((T + 2, H, 128), 9.0, dtype=BF16, device="cuda")
    lens_t = X.lens.clone()
    call = lambda: cache.attention_f8(q, X.kp, X.vp, X.ks, X.vs, table, X.starts, lens_t, out[:T], workspace=ws, **kw)

    def check(L):
        k8, v8 = values(X.kp, X.ks), values(X.vp, X.vs)
        for b, n in enumerate(news):
            if not n:
                continue
            seen = tree_seen(trees[b], L[b], window, sinks) if tree else chain_seen(n, L[b], window, sinks)
            if b == 0:
                seen[:, [j for j in gone if j < L[b]]] = False
            p = torch.arange(L[b], device="cuda")
            page = X.t[b][p // ps].long()
            r = slice(X.st[b], X.st[b] + n)
            check_rows(out[r], *ref_rows(q[r], k8[page, p % ps], v8[page, p % ps], seen), what=f"sequence {b}")
        assert (out[T:] == 9.0).all() and (ws[need:] == 255).all()

    call()
    check(lens)
    first = out.clone()
    call()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for L in ([max(n, x // 3) for n, x in zip(news, lens)], lens):
        lens_t.copy_(ints(L))
        out[:T].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check(L)
    assert torch.equal(out, first)


@pads
@pytest.mark.parametrize("heads", [2, 40, 3600])
def test_masks_that_leave_a_row_empty(heads, pad):
    B = Batch8(14, [3, 3], [3, 40], 16, 1, pad=pad)
    q = rnd(B.g, 6, heads, 128)
    trees = [[{0}, set(), {0, 2}], [set(), {1}, {1, 2}]]
    out = B.attend(q, tree=tree_words(trees, 1))
    assert (out[1] == 0).all()
    B.check(q, out, lambda b: tree_seen(trees[b], B.L[b]))


@pads
@pytest.mark.parametrize("H", [4, 480])
@pytest.mark.parametrize("news,lens,tree", [([1, 1], [70, 3000], False), ([6, 20], [70, 333], True), ([90], [200], False),
                                            ([6, 60], [70, 333], True)])
def test_positions_that_are_not_seen_have_no_part(news, lens, tree, pad, H):
    """Pages' rows behind the sequences' ends, free pages and drafted tokens of other branches hold NaN, free pages scales of NaN too."""
    B = Batch8(15, news, lens, 16, 2, pad=pad)
    used = torch.zeros(B.n_pages, 16, dtype=torch.bool, device="cuda")
    for b, L in enumerate(lens):
        at = torch.arange(L, device="cuda")
        used[B.t[b][at // 16].long(), at % 16] = True
    for p, s in ((B.kp, B.ks), (B.vp, B.vs)):
        p.view(torch.uint8)[~used] = 0x7f
        s.view(torch.uint8)[~used.any(1)] = 255
    rng = random.Random(6)
    trees = [random_tree(rng, n) for n in news]
    if tree:   # a leaf that no one but itself sees
        at = lens[1] - 1
        B.kp.view(torch.uint8)[B.table[1][at // 16], at % 16, 0] = 0xff
        B.vp.view(torch.uint8)[B.table[1][at // 16], at % 16, 1] = 0xff
    q = rnd(B.g, sum(news), H, 128)
    out = B.attend(q, **(dict(tree=tree_words(trees, 1)) if tree else {}))
    B.check(q, out, lambda b: tree_seen(trees[b], lens[b]) if tree else chain_seen(news[b], lens[b]))


@pytest.mark.parametrize("heads", [4, 80, 3600])
def test_seen_values_that_are_not_finite(heads):
    """A NaN in a seen value reaches its dim of the rows that see it, a NaN in a seen key their every dim; a scale of NaN as its rows
    would."""
    B = Batch8(17, [3, 3, 2], [40, 300, 90], 16, 2)
    B.vp.view(torch.uint8)[B.table[0][1], 3, 0, 17] = 0x7f
    B.kp.view(torch.uint8)[B.table[1][2], 5, 1, 99] = 0xff
    B.vs.view(torch.uint8)[B.table[2][3], 0, 1] = 255
    q = rnd(B.g, 8, heads, 128)
    out = B.attend(q)
    h = heads // 2
    assert out[:3, :h, 17].isnan().all() and out[:3].isnan().sum() == 3 * h
    assert out[3:6, h:].isnan().all() and not out[3:6, :h].isnan().any()
    assert out[6:, h:].isnan().all() and not out[6:, :h].isnan().any()


@pads
@pytest.mark.parametrize("heads", [4, 80, 3600])
def test_pages_outside_the_pool_hold_nothing(heads, pad):
    news, lens = [1, 2, 1], [100, 60, 40]
    for ps in (16, 64):
        B = Batch8(16, news, lens, ps, 2, pad=pad)
        table = [list(r) for r in B.table]
        gone = [set(), set(), set()]
        for b, e, value in ((0, 1, -1), (0, 0, B.n_pages), (1, 0, 1 << 30), (2, None, -7)):
            for x in range(len(table[b])) if e is None else [min(e, -(-lens[b] // ps) - 1)]:
                table[b][x] = value
                gone[b] |= set(range(x * ps, (x + 1) * ps))
        q = rnd(B.g, 4, heads, 128)
        out = B.attend(q, table=ints(table))

        def seen(b):
            s = chain_seen(news[b], lens[b])
            s[:, [j for j in gone[b] if j < lens[b]]] = False
            return s
        B.check(q, out, seen)
        assert (out[3] == 0).all()


@pads
@pytest.mark.parametrize("H", [4, 40, 2600])
def test_rows_behind_the_last_sequence_stay(H, pad):
    """A padded batch: more rows than tokens, output rows and columns beyond the call's left as they were, queries as views."""
    B = Batch8(18, [2, 5], [100, 37], 16, 2, pad=pad)
    wide = rnd(B.g, 12, H + 3, 128)
    q = wide[:, 1:1 + H]
    out = torch.full((12, H + 1, 128), 9.0, dtype=BF16, device="cuda")
    B.attend(q, out=out[:, :H], max_rows=5, max_keys=100)
    B.check(q, out[:, :H], lambda b: chain_seen(B.news[b], B.L[b]))
    assert (out[7:] == 9.0).all() and (out[:, H:] == 9.0).all()


@pytest.mark.parametrize("H", [4, 3200])
@pytest.mark.parametrize("starts,lens", [([0, 3, 1, 4], [50, 50, 50]), ([-1, 2, 3, 4], [50, 50, 50]), ([0, 1, 2, 4], [-5, 50, 1 << 30]),
                                         ([0, 1, 2, 1 << 30], [50, 2000000000, 0])])
def test_senseless_numbers_do_nothing_outside(starts, lens, H):
    """Starts that do not ascend, negative and huge lengths: whatever rows come out, nothing outside the tensors is touched."""
    B = Batch8(19, [1, 1, 2], [50, 50, 50], 16, 2)
    pool = torch.cat([x.view(torch.uint8).flatten() for x in (B.kp, B.vp, B.ks, B.vs)])
    q, k, v = rnd(B.g, 4, H, 128), rnd(B.g, 4, 2, 128), rnd(B.g, 4, 2, 128)
    out = torch.full((6, H, 128), 9.0, dtype=BF16, device="cuda")
    cache.attention_f8(q, B.kp, B.vp, B.ks, B.vs, B.t, ints(starts), ints(lens), out[:4])
    cache.attention_f8(q, B.kp, B.vp, B.ks, B.vs, B.t, ints(starts), ints(lens), out[:4], max_rows=1, max_keys=20)
    assert (out[4:] == 9.0).all()
    assert torch.equal(pool, torch.cat([x.view(torch.uint8).flatten() for x in (B.kp, B.vp, B.ks, B.vs)]))
    cache.append_f8(q, k, v, B.kp, B.vp, B.ks, B.vs, B.t, ints(starts), ints(lens), out[:4], table_kind=ops.TABLE_NONE)
    assert (out[4:] == 9.0).all()


@pytest.mark.parametrize("scale", [0.02, 1.0])
@pytest.mark.parametrize("n", [1, 40])
def test_scales_and_large_scores(scale, n):
    """Scores far from zero, rising along the keys, so that the references are raised again and again."""
    B = Batch8(20, [n], [900], 32, 2)
    e = exps(B.ks)
    at = torch.arange(29, device="cuda")
    e[B.t[0][:29].long()] += (at // 10)[:, None, None].int()
    B.ks = scales_of(e)
    q = rnd(B.g, n, 8, 128)
    out = B.attend(q, scale=scale)
    B.check(q, out, lambda b: chain_seen(n, 900), scale)


@pytest.mark.parametrize("scale", [0.02, 1.0])
@pytest.mark.parametrize("H,HK,n,L", [(128, 8, 290, 4500), (14, 2, 300, 1300), (64, 8, 200, 1000), (40, 2, 600, 1300)])
def test_large_scores_of_chunks(H, HK, n, L, scale):
    """The same of many rows: rows whose sums grow take higher references, in the middle of a block and of its parts."""
    B = Batch8(30, [n], [L], 32, HK)
    e = exps(B.ks)
    pages = -(-L // 32)
    e[B.t[0][:pages].long()] += (torch.arange(pages, device="cuda") * 6 // pages)[:, None, None].int()
    B.ks = scales_of(e)
    q = rnd(B.g, n, H, 128)
    out = B.attend(q, scale=scale)
    at = [0, 1, n // 2, n - 1]
    k, v = B.rows(0)
    check_rows(out[at], *ref_rows(q[at], k, v, chain_seen(n, L)[at], scale), what="rows")


def test_far_pages():
    """Pages whose offsets pass 32 bits, interleaved keys and values, scales side by side in one buffer."""
    pages, ps, HK = 10, 16, 2
    stride = (1 << 29) + 4096
    big = torch.zeros(9 * stride + 2 * ps * HK * 128, dtype=torch.uint8, device="cuda")
    kp, vp = (big.as_strided((pages, ps, HK, 128), (stride, 2 * HK * 128, 128, 1), o).view(F8) for o in (0, HK * 128))
    sc = torch.zeros(pages, 2, 1, HK, dtype=torch.uint8, device="cuda").view(E8)
    B = Batch8(21, [1, 3], [70, 33], ps, HK, pages=pages)
    kp.view(torch.uint8).copy_(B.kp.view(torch.uint8))
    vp.view(torch.uint8).copy_(B.vp.view(torch.uint8))
    sc.view(torch.uint8)[:, 0], sc.view(torch.uint8)[:, 1] = B.ks.view(torch.uint8), B.vs.view(torch.uint8)
    q = rnd(B.g, 4, 6, 128)
    want = B.attend(q)
    assert torch.equal(cache.attention_f8(q, kp, vp, sc[:, 0], sc[:, 1], B.t, B.starts, B.lens), want)
    B.check(q, want, lambda b: chain_seen(B.news[b], B.L[b]))
    k, v = rnd(B.g, 4, HK, 128), rnd(B.g, 4, HK, 128)
    for p in ((B.kp, B.vp, B.ks, B.vs), (kp, vp, sc[:, 0], sc[:, 1])):
        cache.append_f8(None, k, v, *p, B.t, B.starts, B.lens, table_kind=ops.TABLE_NONE)
    for x, y in ((kp, B.kp), (vp, B.vp), (sc[:, 0], B.ks), (sc[:, 1], B.vs)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("H", [6, 30])
def test_far_pages_of_chunks(H):
    """The same of a chunk and a single token beside it; of many heads in the kernel of many rows."""
    pages, ps, HK = 8, 256, 2
    stride = (1 << 31) + 4096
    big = torch.zeros(7 * stride + 2 * ps * HK * 128, dtype=torch.uint8, device="cuda")
    kp, vp = (big.as_strided((pages, ps, HK, 128), (stride, 2 * HK * 128, 128, 1), o).view(F8) for o in (0, HK * 128))
    B = Batch8(27, [600, 1], [1100, 300], ps, HK, pages=pages)
    kp.view(torch.uint8).copy_(B.kp.view(torch.uint8))
    vp.view(torch.uint8).copy_(B.vp.view(torch.uint8))
    q = rnd(B.g, 601, H, 128)
    want = B.attend(q)
    assert torch.equal(cache.attention_f8(q, kp, vp, B.ks, B.vs, B.t, B.starts, B.lens), want)
    for b, at in ((0, [0, 300, 599]), (1, [0])):
        k, v = B.rows(b)
        check_rows(want[[B.st[b] + i for i in at]], *ref_rows(q[[B.st[b] + i for i in at]], k, v, chain_seen(B.news[b], B.L[b])[at]))


@pytest.mark.parametrize("H", [2, 80])
def test_tokens_before_the_first_position(H):
    """More tokens than positions: those before the first see nothing, and have no place in the pages."""
    B = Batch8(28, [40, 3], [25, 70], 16, 2)
    q = rnd(B.g, 43, H, 128)
    out = torch.full((43, H, 128), 9.0, dtype=BF16, device="cuda")
    B.attend(q, out=out)
    assert (out[:15] == 0).all()
    seen = chain_seen(25, 25)
    k, v = B.rows(0)
    check_rows(out[15:40], *ref_rows(q[15:40], k, v, seen), what="the rest")
    k, v = rnd(B.g, 43, 2, 128), rnd(B.g, 43, 2, 128)
    kp, vp, ks, vs = (x.clone() for x in (B.kp, B.vp, B.ks, B.vs))
    q_out = torch.full((43, H, 128), 9.0, dtype=BF16, device="cuda")
    cache.append_f8(q, k, v, B.kp, B.vp, B.ks, B.vs, B.t, B.starts, B.lens, q_out, table_kind=ops.TABLE_NONE)
    assert (q_out[:15] == 9.0).all() and not (q_out[15:] == 9.0).all((1, 2)).any()
    cache.append_f8(q[15:], k[15:], v[15:], kp, vp, ks, vs, B.t, ints([0, 25, 28]), B.lens, table_kind=ops.TABLE_NONE)
    for x, y in ((kp, B.kp), (vp, B.vp), (ks, B.ks), (vs, B.vs)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("H,n,rows,L", [(16, 9, 7, 500), (128, 300, 290, 4500)])
def test_more_tokens_than_the_call_is_sized_for(H, n, rows, L):
    B = Batch8(29, [n], [L], 32, 8)
    q = rnd(B.g, n, H, 128)
    out = torch.full((n, H, 128), 9.0, dtype=BF16, device="cuda")
    B.attend(q, out=out, max_rows=rows, max_keys=L)
    at = [0, rows // 2, rows - 1]
    k, v = B.rows(0)
    check_rows(out[at], *ref_rows(q[at], k, v, chain_seen(n, L)[at]), what="rows")
    assert (out[rows:] == 9.0).all()


# ------------------------------------------------------------------------------------------------ append
def angles(n):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    return a.cos().float().cuda(), a.sin().float().cuda()


def turned(x, w, table, pos, pairing=0, rot=128, eps=1e-6):
    """Norm and rotation in 64 bits, and a bound of what fp32 may be off by: the norm's factor is a sum of 128 squares (2^-18 with the
    root and two products), a rotated dim the sum of two products of up to |x0| + |x1| with two roundings more."""
    y = x.double() / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    mag = y.abs()
    if table is not None:
        c, s = (t[pos].double()[:, None, :rot // 2] for t in table)
        i = torch.arange(rot // 2, device=x.device)
        a, b = (2 * i, 2 * i + 1) if pairing == 0 else (i, i + rot // 2)
        z = y.clone()
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
        mag[..., a] = mag[..., b] = mag[..., a] + mag[..., b]
        y = z
    return y, mag * 2.0 ** -17


def plain_append(B, x, off, pages, scales, live=None):
    """Rows x [T, HK, 128] (fp64, off by up to `off`) into copies of pages and scales, by the definition; returns the exponents, and
    which bytes and scales they allow: (pages that hold x - off and x + off, their scales) at each border."""
    out = []
    for sign in (-1, 1):
        p, e = pages.clone(), exps(scales)
        for b, n in enumerate(B.news):
            c, t0 = B.L[b] - n, B.st[b]
            slots = [(s, t0 + s - c) for s in range(max(c, 0), B.L[b]) if live is None or live[t0 + s - c]]
            for g in sorted({s // GROUP for s, _ in slots}):
                page = B.table[b][g * GROUP // B.ps]
                if not 0 <= page < B.n_pages:
                    continue
                r0, at = g * GROUP % B.ps, [(s, t) for s, t in slots if s // GROUP == g]
                y = x[[t for _, t in at]]
                y = y + sign * off[[t for _, t in at]] * y.sign()
                new = exponent(torch.where(torch.isfinite(y), y.abs(), 0.0).amax((0, 2)))
                first = max(c, g * GROUP) - g * GROUP
                if first:
                    old = e[page, r0 // GROUP].clone()
                    new = torch.maximum(new, old)
                    q = p[page, r0:r0 + first].float().double() * torch.exp2((old - new).double())[:, None]
                    p[page, r0:r0 + first] = to_f8(q)
                e[page, r0 // GROUP] = new.to(e.dtype)
                for (s, t), row in zip(at, y):
                    p[page, s % B.ps] = to_f8(row * torch.exp2(-new.double())[:, None])
        out.append((p, scales_of(e)))
    return out


def check_append(B, x, off, before, got, live=None):
    (lo, slo), (hi, shi) = plain_append(B, x, off, before[0], before[1], live)
    g, a, b = (t.view(torch.uint8).int() for t in (got[1], slo, shi))
    assert ((g == a) | (g == b)).all(), "scales"
    w, a, b = values(*got), values(lo, slo), values(hi, shi)
    assert torch.equal(w.isnan(), a.isnan())
    bits = got[0].view(torch.uint8)
    same = (bits == lo.view(torch.uint8)) | (bits == hi.view(torch.uint8)) | w.isnan()   # (a NaN of either sign: which has no meaning)
    # (a byte between the two only where the errors' bound spans a whole step, or the two borders' scales differ)
    inside = (w >= torch.minimum(a, b)) & (w <= torch.maximum(a, b))
    assert (same | inside).all(), f"{int((~(same | inside)).sum())} bytes differ"


# tokens of each sequence, lengths, heads, kv heads, page size, by_head
APPENDS = [
    ([1], [1], 1, 1, 16, False),
    ([1], [17], 4, 2, 16, False),                       # a group of its own
    ([1, 1, 1, 1], [16, 32, 15, 2], 4, 4, 32, False),   # into groups that hold rows
    ([2, 0, 16, 17], [33, 5, 16, 50], 6, 2, 16, True),
    ([40, 1, 33], [40, 130, 100], 8, 1, 64, False),
    ([300], [517], 3, 3, 128, True),
    ([1] * 70, [1 + 3 * i for i in range(70)], 2, 1, 16, False),
    ([5, 31] * 20, [9, 40] * 20, 5, 5, 256, False),
]


@pytest.mark.parametrize("c", APPENDS, ids=lambda c: f"{len(c[0])}seq{max(c[0])}of{max(c[1])}h{c[2]}g{c[3]}p{c[4]}")
@pytest.mark.parametrize("loud", [0.01, 30.0])
def test_append(c, loud):
    """Against the restatement: bits of the values, what fp32 allows of the keys; groups that grow (loud) and that do not. Queries as the
    bf16 append's, bit for bit."""
    news, lens, H, HK, ps, by_head = c
    B = Batch8(31, news, lens, ps, HK, by_head)
    T = sum(news)
    qkv = rnd(B.g, T, H + 2 * HK, 128)
    q, k, v = qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:] * torch.tensor(loud, dtype=BF16, device="cuda")
    qw, kw = (torch.rand(128, generator=B.g, device="cuda") + 0.5 for _ in range(2))
    kw = kw * loud
    tab = angles(max(lens))
    was = [x.clone() for x in (B.kp, B.ks, B.vp, B.vs)]
    out = cache.append_f8(q, k, v, B.kp, B.vp, B.ks, B.vs, B.t, B.starts, B.lens, q_norm=qw, k_norm=kw, table=tab)
    pos = torch.cat([torch.arange(L - n, L) for n, L in zip(news, lens)]).cuda()
    y, off = turned(k, kw, tab, pos)
    check_append(B, y, off, was[:2], (B.kp, B.ks))
    check_append(B, v.double(), torch.zeros_like(v.double()), was[2:], (B.vp, B.vs))
    kp, vp = (torch.zeros(B.n_pages, ps, HK, 128, dtype=BF16, device="cuda") for _ in range(2))
    assert torch.equal(out, cache.append(q, k, v, kp, vp, B.t, B.starts, B.lens, q_norm=qw, k_norm=kw, table=tab))


@pytest.mark.parametrize("kind,pairing,rot", [(ops.TABLE_NONE, 0, 128), (ops.TABLE_COSSIN_F32, 1, 128), (ops.TABLE_COSSIN_F32, 1, 32),
                                              (ops.TABLE_COSSIN_F32, 0, 50), (ops.TABLE_MAT2_F32, 1, 96), (ops.TABLE_MAT2_BF16, 0, 128)])
def test_append_rotations(kind, pairing, rot):
    """Every table kind and pairing, table rows from `positions`; tokens whose row is not one of the table's are left out whole."""
    B = Batch8(32, [21, 3], [50, 3], 32, 2)
    T, n = 24, 60
    q, k, v = rnd(B.g, T, 3, 128), rnd(B.g, T, 2, 128), rnd(B.g, T, 2, 128)
    c, s = angles(n)
    pos = torch.randint(0, n, (T,), generator=B.g, device="cuda")
    bad = torch.zeros(T, dtype=torch.bool, device="cuda")
    if kind != ops.TABLE_NONE:
        pos[[4, 22]] = torch.tensor([n, -1], device="cuda")
        bad[[4, 22]] = True
        k[bad], v[bad] = 1000.0, 1000.0
    if kind in (ops.TABLE_MAT2_F32, ops.TABLE_MAT2_BF16):
        m = torch.stack([c, -s, s, c], -1)[:, :rot // 2].flatten(1)
        if kind == ops.TABLE_MAT2_BF16:
            m = m.to(BF16)
            c, s = m.view(n, -1, 4)[..., 3].float(), m.view(n, -1, 4)[..., 2].float()
        table = (m.contiguous(), None)
    else:
        table = (c, s)
    was = [x.clone() for x in (B.kp, B.ks, B.vp, B.vs)]
    out = torch.full((T, 3, 128), 7.0, dtype=BF16, device="cuda")
    cache.append_f8(q, k, v, B.kp, B.vp, B.ks, B.vs, B.t, B.starts, B.lens, out, table_kind=kind,
                    table=None if kind == ops.TABLE_NONE else table, positions=pos.int(), pairing=pairing, rot=rot)
    y, off = turned(k, None, None if kind == ops.TABLE_NONE else (c, s), pos.clamp(0, n - 1), pairing, rot)
    live = (~bad).tolist()
    check_append(B, y, off, was[:2], (B.kp, B.ks), live)
    check_append(B, v.double(), torch.zeros_like(v.double()), was[2:], (B.vp, B.vs), live)
    assert (out[bad] == 7.0).all() and not (out[~bad] == 7.0).all()


def test_append_of_values_that_are_not_finite():
    """Infinities and NaN are held as NaN and leave the scale to the others; zeros, the smallest and the largest values."""
    B = Batch8(33, [16, 3, 1, 2], [16, 20, 32, 18], 16, 1)
    v = rnd(B.g, 22, 1, 128)
    v[3, 0, 5], v[4, 0, 6], v[17, 0, 7] = float("nan"), float("inf"), -float("inf")
    v[19] = 0.0
    v[20] = 3.0e38
    v[21] = 1.0e-38
    was = [x.clone() for x in (B.vp, B.vs)]
    cache.append_f8(None, v, v, B.kp, B.vp, B.ks, B.vs, B.t, B.starts, B.lens, table_kind=ops.TABLE_NONE)
    check_append(B, v.double(), torch.zeros_like(v.double()), was, (B.vp, B.vs))
    assert B.kp.view(torch.uint8)[B.table[0][0], 3].eq(0x7f).logical_or(B.kp.view(torch.uint8)[B.table[0][0], 3].eq(0xff)).all()   # (its norm is NaN)


def test_append_token_by_token_holds_what_one_call_does():
    """A sequence appended one token at a time: each value within the roundings of its group's scales so far, the scales those of one call."""
    B = Batch8(34, [100], [100], 32, 3)
    v = rnd(B.g, 100, 3, 128) * torch.exp2(torch.randint(-6, 6, (100, 1, 1), generator=B.g, device="cuda")).to(BF16)
    one = [x.clone() for x in (B.kp, B.vp, B.ks, B.vs)]
    cache.append_f8(None, v, v, *one, B.t, ints([0, 100]), ints([100]), table_kind=ops.TABLE_NONE)
    for i in range(100):
        cache.append_f8(None, v[i:i + 1], v[i:i + 1], B.kp, B.vp, B.ks, B.vs, B.t, ints([0, 1]), ints([i + 1]), table_kind=ops.TABLE_NONE)
    B.L = [100]
    page = B.t[0].long()
    assert torch.equal(B.vs.view(torch.uint8)[page[:3]], one[3].view(torch.uint8)[page[:3]])
    d = (B.rows(0)[1] - v.double()).abs()
    top = torch.exp2(exps(B.vs).double())[page].flatten(0, 1).repeat_interleave(GROUP, 0)[:100, :, None]
    # half a step of e4m3 once, and 2^-10 of the scale for each time the group grew (at most 12 octaves) where the value is subnormal
    assert (d <= 2.0 ** -4 * v.double().abs() + 12 * 2.0 ** -10 * top).all()


@pytest.mark.parametrize("B", [1, 3, 90])
def test_append_of_sequences_that_begin_late(B):
    """Rows before the first sequence are left out: the search for a group's sequence begins behind its first numbers."""
    b = Batch8(36, [17] * B, [40] * B, 16, 2)
    v, lead = rnd(b.g, 200 + 17 * B, 2, 128), 150
    want = [x.clone() for x in (b.kp, b.vp, b.ks, b.vs)]
    cache.append_f8(None, v[lead:], v[lead:], *want, b.t, b.starts, b.lens, table_kind=ops.TABLE_NONE)
    cache.append_f8(None, v, v, b.kp, b.vp, b.ks, b.vs, b.t, b.starts + lead, b.lens, table_kind=ops.TABLE_NONE)
    for x, y in zip((b.kp, b.vp, b.ks, b.vs), want):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_append_leaves_the_rest():
    """Rows behind the sequences, pages of others and their scales, queries' columns of others; a page that the pool does not have."""
    B = Batch8(35, [3, 20], [21, 20], 16, 2)
    k = rnd(B.g, 30, 2, 128)
    table = [list(r) for r in B.table]
    lost = table[1][1]
    table[1][1] = B.n_pages
    touched = torch.zeros(B.n_pages, 16, dtype=torch.bool, device="cuda")
    for b in (0, 1):
        at = torch.arange(B.L[b], device="cuda")
        touched[B.t[b][at // 16].long(), at % 16] = True
    touched[lost] = False
    touched[B.table[0][0]] = False
    was = [x.view(torch.uint8).clone() for x in (B.kp, B.vp, B.ks, B.vs)]
    cache.append_f8(None, k, k, B.kp, B.vp, B.ks, B.vs, ints(table), B.starts, B.lens, table_kind=ops.TABLE_NONE)
    now = [x.view(torch.uint8) for x in (B.kp, B.vp, B.ks, B.vs)]
    for i in (0, 1):
        assert torch.equal(now[i][~touched], was[i][~touched])
        assert torch.equal(now[2 + i][~touched.any(1)], was[2 + i][~touched.any(1)])
        assert not torch.equal(now[i][touched], was[i][touched])


# ------------------------------------------------------------------------------------------------ copies, and all together
@pytest.mark.parametrize("layers", [None, 3])
@pytest.mark.parametrize("by_head", [False, True, None])
def test_copy_pages(layers, by_head):
    """Pages and their scales, token by token, head by head, and rows apart from each other; pairs outside the pool are left out."""
    n, ps, HK = 9, 32, 3
    g = gen(41)
    L = (layers,) if layers else ()
    shape = L + ((n, HK, ps, 128) if by_head else (n, ps, HK, 128 if by_head is not None else 256))

    def pool():
        t = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
        return (t.transpose(-3, -2) if by_head else t[..., :128] if by_head is None else t).view(F8)
    kp, vp = pool(), pool()
    if by_head is None:   # (heads 256 bytes apart)
        assert kp.stride(-2) == 256
    ks, vs = (torch.randint(0, 256, L + (n, 2, HK), generator=g, device="cuda", dtype=torch.uint8).view(E8) for _ in range(2))
    all_ = [x.view(torch.uint8) for x in (kp, vp, ks, vs)]
    want = [x.clone() for x in all_]
    src, dst = [0, 0, 7, 3, 99], [4, 5, 2, -1, 6]
    for x in want:
        x = x if layers else x[None]
        for a, b in zip(src[:3], dst[:3]):
            x[:, b] = x[:, a]
    cache.copy_pages_f8(kp, vp, ks, vs, ints(src), ints(dst))
    for x, y in zip(all_, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("tree", [False, True])
def test_a_serving_loop(tree):
    """Prompts appended and attended, single tokens, a fork with its last page copied, drafted tokens (a tree: its accepted branch
    appended again), each step's attention against what the pages hold, the pages against the tokens' rows; the decode step captured
    and replayed."""
    ps, HK, H = 16, 2, 8
    rng, g = random.Random(9), gen(51)
    n_pages = 64
    pool = cache.PagePool(n_pages)
    B = Batch8(52, [0], [0], ps, HK, pages=n_pages)
    P = (B.kp, B.vp, B.ks, B.vs)
    tables = [pool.alloc(3), pool.alloc(2)]
    truth = [torch.zeros(0, HK, 128, device="cuda") for _ in range(2)]   # the values' rows

    def step(news, lens, mask=None, positions=None, keep=True):
        T = sum(news)
        q, k, v = rnd(g, T, H, 128), rnd(g, T, HK, 128), rnd(g, T, HK, 128)
        width = max(len(t) for t in tables)
        t = ints([list(x) + [-1] * (width - len(x)) for x in tables])
        st = [0]
        for n in news:
            st.append(st[-1] + n)
        qo = cache.append_f8(q, k, v, *P, t, ints(st), ints(lens), table=angles(200), positions=positions)
        out = cache.attention_f8(qo, *P, t, ints(st), ints(lens), max_rows=max(news), max_keys=max(lens),
                                 tree=None if mask is None else tree_words(mask, 1))
        kv, vv = values(B.kp, B.ks), values(B.vp, B.vs)
        for b, n in enumerate(news):
            at = torch.arange(lens[b], device="cuda")
            page, row = t[b][at // ps].long(), at % ps
            seen = tree_seen(mask[b], lens[b]) if mask else chain_seen(n, lens[b])
            check_rows(out[st[b]:st[b + 1]], *ref_rows(qo[st[b]:st[b + 1]], kv[page, row], vv[page, row], seen), what=f"sequence {b}")
            rows = torch.cat([truth[b][:lens[b] - n], v[st[b]:st[b + 1]].float()])
            d, top = (vv[page, row] - rows).abs(), torch.exp2(exps(B.vs)[page, row // GROUP].double())[..., None]
            assert (d <= 2.0 ** -4 * rows.abs() + 2.0 ** -7 * top).all()   # (a few groups grew an octave or two: 2^-10 of the scale each)
            if keep:
                truth[b] = rows
        return q, k, v, st

    lens = [37, 20]
    step([37, 20], lens)
    for _ in range(3):
        lens = [x + 1 for x in lens]
        step([1, 1], lens)
    # a third sequence forks the first: the full pages shared, the last one its own
    tables.append(pool.fork(tables[0]))
    truth.append(truth[0].clone())
    pair = pool.own(tables[2], 2)
    cache.copy_pages_f8(*P, ints([pair[0]]), ints([pair[1]]))
    lens = [lens[0] + 1, lens[1] + 1, lens[0] + 1]
    step([1, 1, 1], lens)
    if tree:
        n = [7, 4, 6]
        for i, t in enumerate(tables):
            t += pool.alloc(-(-(lens[i] + 7) // ps) - len(t))
        trees = [random_tree(rng, x) for x in n]
        ctx = lens
        depth = torch.tensor([c + len(s) - 1 for c, t in zip(ctx, trees) for s in t], dtype=torch.int32, device="cuda")
        q, k, v, st = step(n, [a + b for a, b in zip(ctx, n)], trees, depth, keep=False)
        # the branch of the last drafted token is accepted
        take = [sorted(t[-1]) for t in trees]
        at = torch.tensor([st[b] + x for b in range(3) for x in take[b]], device="cuda")
        s2 = [0]
        for x in take:
            s2.append(s2[-1] + len(x))
        lens = [c + len(x) for c, x in zip(ctx, take)]
        width = max(len(t) for t in tables)
        cache.append_f8(None, k[at], v[at], *P, ints([list(x) + [-1] * (width - len(x)) for x in tables]), ints(s2), ints(lens),
                        table=angles(200))
        for b in range(3):
            truth[b] = torch.cat([truth[b], v[at[s2[b]:s2[b + 1]]].float()])
        for i, t in enumerate(tables):
            t += pool.alloc(max(0, -(-(lens[i] + 1) // ps) - len(t)))
        lens = [x + 1 for x in lens]
        step([1, 1, 1], lens)


def test_a_captured_step():
    """Append and attention of a decode step captured, replayed over other lengths and tokens, against eager calls, bit for bit."""
    ps, HK, H, n = 16, 2, 8, 3
    g = gen(61)
    B = Batch8(62, [1] * n, [90, 200, 40], ps, HK)
    P = (B.kp, B.vp, B.ks, B.vs)
    q, k, v = rnd(g, n, H, 128), rnd(g, n, HK, 128), rnd(g, n, HK, 128)
    qo, out = torch.empty_like(q), torch.empty_like(q)
    lens, tab = B.lens.clone(), angles(300)
    ws = torch.empty(max(256, cache.attention_f8_ws_bytes(n, n, 1, 208, H, HK, ps)), dtype=torch.uint8, device="cuda")

    def call():
        cache.append_f8(q, k, v, *P, B.t, B.starts, lens, qo, table=tab)
        cache.attention_f8(qo, *P, B.t, B.starts, lens, out, max_rows=1, max_keys=208, workspace=ws)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for L in ([88, 199, 33], [90, 208, 48], [1, 17, 16], [88, 199, 33]):
        lens.copy_(ints(L))
        for t, x in ((q, H), (k, HK), (v, HK)):
            t.copy_(rnd(g, n, x, 128))
        saved = [x.view(torch.uint8).clone() for x in P]
        graph.replay()
        torch.cuda.synchronize()
        got = [out.clone(), *(x.view(torch.uint8).clone() for x in P)]
        for x, y in zip(P, saved):
            x.view(torch.uint8).copy_(y)
        call()
        for x, y in zip(got, [out, *(x.view(torch.uint8) for x in P)]):
            assert torch.equal(x, y)
        for b in range(n):
            at = torch.arange(L[b], device="cuda")
            page = B.t[b][at // ps].long()
            check_rows(out[b:b + 1], *ref_rows(qo[b:b + 1], values(B.kp, B.ks)[page, at % ps], values(B.vp, B.vs)[page, at % ps],
                                               chain_seen(1, L[b])), what=f"sequence {b}")


def test_another_stream_and_a_workspace_of_ones_own():
    B = Batch8(71, [1, 1], [9000, 500], 16, 1)
    q = rnd(B.g, 2, 4, 128)
    want = B.attend(q, max_rows=1, max_keys=9000)
    need = cache.attention_f8_ws_bytes(2, 2, 1, 9000, 4, 1, 16)
    assert need > 0
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = B.attend(q, max_rows=1, max_keys=9000, workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and (ws[need:] == 255).all()
    with pytest.raises(ValueError):
        B.attend(q, max_rows=1, max_keys=9000, workspace=ws[:need - 1])


def test_refusals_by_name():
    B = Batch8(72, [1], [20], 16, 2)
    q, k = rnd(B.g, 1, 4, 128), rnd(B.g, 1, 2, 128)
    bf = torch.zeros(4, 16, 2, 128, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        cache.attention_f8(q, bf, bf, B.ks, B.vs, B.t, B.starts, B.lens)
    with pytest.raises(ValueError, match="float8_e8m0fnu"):
        cache.attention_f8(q, B.kp, B.vp, B.ks.view(torch.uint8), B.vs, B.t, B.starts, B.lens)
    with pytest.raises(ValueError, match="float8_e8m0fnu"):
        cache.append_f8(None, k, k, B.kp, B.vp, B.ks[1:], B.vs[1:], B.t, B.starts, B.lens, table_kind=ops.TABLE_NONE)
    with pytest.raises(ValueError, match="table required"):
        cache.append_f8(None, k, k, B.kp, B.vp, B.ks, B.vs, B.t, B.starts, B.lens)
    with pytest.raises(ValueError, match="of different lengths"):
        cache.copy_pages_f8(B.kp, B.vp, B.ks, B.vs, ints([1]), ints([2, 3]))
    with pytest.raises(_lib.LrError):
        cache.attention_f8(q, B.kp, B.vp, B.ks, B.vs, B.t, B.starts, B.lens, window=-1)
    empty = torch.empty(0, 4, 128, dtype=BF16, device="cuda")
    assert cache.attention_f8(empty, B.kp, B.vp, B.ks, B.vs, B.t, B.starts, B.lens).shape == (0, 4, 128)
