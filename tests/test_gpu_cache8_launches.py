"""attention_f8's launches of large batches, and those that are cut because a workgroup holds so many page-table entries (which these are:
tests/test_cache8_launches.py), against a 64-bit attention over what the pages hold."""
from __future__ import annotations

import random

import pytest
import torch

from localrouter_amd import cache
from tests.cache8_util import values
from tests.cache_util import HALF, ref_rows, rnd
from tests.launch_util import LAUNCHES8
from tests.test_gpu_cache import chain_seen, ints, random_tree, tree_words
from tests.test_gpu_cache8 import BF16, Batch8

pytestmark = pytest.mark.gpu


def tree_seen(sets, L):
    c = L - len(sets)
    seen = torch.zeros(len(sets), L, dtype=torch.bool)
    seen[:, :c] = True
    for i, s in enumerate(sets):
        seen[i, [c + x for x in s]] = True
    return seen


def check_long(got, ref, mag, keys, what):
    """cache_util's tolerance, of four times its queries (scores that a few keys of tens of thousands dominate, or a part left out would
    not show): |q k| below 2^10 in all, 2^-10 of p_j above and below the fraction bar, and two sums of `keys` terms."""
    got = got.double().cpu()
    tol = HALF * ref.abs() + (2 * HALF + 2.0 ** -9 + 2 * keys * 2.0 ** -24) * mag + 1e-30
    d = (got - ref).abs()
    assert (d <= tol).all(), f"{what}: {int((d > tol).sum())} values off, worst {float((d / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("sizes", [s for s, _ in LAUNCHES8], ids=str)
def test_launches(sizes, tree):
    """Most sequences short, one as long as the call is sized for, some longer, one without tokens, one at the first part's end; a page that
    the pool does not have, NaN behind the sequences; bit for bit again in the same workspace, nothing behind it touched; other lengths at a
    replay."""
    B, rows, most, H, HK, ps = sizes
    rng = random.Random(B + rows)
    if tree and rows > 64:
        rows_of = [64] * B   # (a word a token)
    else:
        rows_of = [rows] + [rng.randrange(0, rows + 1) for _ in range(B - 1)]
    lens = [most] + [rng.randrange(rows, 400) for _ in range(B - 1)]
    if B > 4:
        rows_of[1], rows_of[2], rows_of[3] = 0, rows, rows
        lens[2] = min(most, (61440 if most > 61440 else 16384) + 1)
        lens[3] = rows
    X = Batch8(91, rows_of, lens, ps, HK)
    used = torch.zeros(X.n_pages, ps, dtype=torch.bool, device="cuda")
    for b, L in enumerate(lens):
        at = torch.arange(L, device="cuda")
        used[X.t[b][at // ps].long(), at % ps] = True
    X.kp.view(torch.uint8)[~used], X.vp.view(torch.uint8)[~used] = 0x7f, 0xff
    table = X.t.clone()
    gone = list(range(3 * ps, 4 * ps))
    table[0, 3] = X.n_pages + 1
    T = sum(rows_of)
    trees = [random_tree(rng, n) for n in rows_of]
    kw = dict(max_rows=rows, max_keys=most, tree=tree_words(trees, 1) if tree else None)
    need = cache.attention_f8_ws_bytes(B, T, rows, most, H, HK, ps)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    q = 4 * rnd(X.g, T, H, 128)
    out = torch.full((T + 2, H, 128), 9.0, dtype=BF16, device="cuda")
    lens_t = X.lens.clone()
    call = lambda: cache.attention_f8(q, X.kp, X.vp, X.ks, X.vs, table, X.starts, lens_t, out[:T], workspace=ws, **kw)

    def check(L):
        for b, n in enumerate(rows_of):
            if not n or (b > 5 and b % 17 and b != B - 1):
                continue
            at = sorted({0, n // 2, n - 1})
            seen = (tree_seen(trees[b], L[b]) if tree else chain_seen(n, L[b]))[at]
            seen[:, most:] = False   # (positions beyond max_keys are not seen)
            if b == 0:
                seen[:, [j for j in gone if j < L[b]]] = False
            pages = X.t[b][:-(-L[b] // ps)].long()
            k, v = (values(x[pages], s[pages]).flatten(0, 1)[:L[b]]
                    for x, s in ((X.kp, X.ks), (X.vp, X.vs)))
            r = [X.st[b] + i for i in at]
            check_long(out[r], *ref_rows(q[r], k, v, seen), L[b], f"sequence {b}")
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
    for L in ([max(n, x // 3) for n, x in zip(rows_of, lens)], lens):
        lens_t.copy_(ints(L))
        out[:T].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check(L)
    assert torch.equal(out, first)
