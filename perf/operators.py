"""The cache in pages and the attention over it, and windowed attention over rows, as cases that can be timed and compared.

  window   ops.attention_window: query i at position p = p0 + i, frame f = p // frame, sees key j when j < keys,
           j // frame <= f and (j // frame > f - window or j < sinks); out_i = softmax(scale * q_i k_j) v_j over those keys
  append   cache.append: token t of sequence b takes slot s = lens[b] - n_b + (t - starts[b]) of its sequence (n_b of the
           tokens are sequence b's, lens[b] counts them); per head y = x / sqrt(mean(x^2) + eps) * w, pairs rotated by the
           table row of the token's position; q to rows, k and v to row s % page_size of page page_table[b][s // page_size]
  attend   cache.attention: the tokens of each sequence over its pages. The token of slot p sees j <= p; drafted tokens
           under a tree see the context j < c = lens[b] - n_b and the drafted keys c + x whose bit x is set in the token's
           mask; with a window of n positions, context further back than that and not among the sinks is left out
  copy     cache.copy_pages: pages copied inside the pool, in every layer
  move     cache.move_rows: rows of a sequence moved to other positions of it, in every layer

  listed()             the named cases
  draw(rng)            one more case of the same ranges
  prepare(case, seed)  the inputs and what a program keeps between calls (pools, page tables, output buffers)
  run(state)           one pass; returns its outputs
  work(case)           the bytes and floating-point operations the pass cannot do without
  exact(case, seed)    the outputs in 64 bits

`own` false: plain torch operations in fp32; `own` true: the library's calls.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128
EPS = 1e-6
SCALE = 1.0 / math.sqrt(128.0)
THETA = 10000.0
BF16 = torch.bfloat16


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one new token over the rows of a short prompt: a window of 1,024 tokens behind 4 first tokens
        dict(name="window-token", kind="window", queries=1, keys=1500, p0=1499, heads=32, kv_heads=8, window=1024, sinks=4,
             frame=1),
        # a text encoder's chunk behind 1,777 positions, an odd length
        dict(name="window-text-2319", kind="window", queries=2319, keys=4096, p0=1777, heads=32, kv_heads=8, window=1024,
             sinks=4, frame=1),
        # autoregressive video: 16 frames of 32 x 32 tokens, each over its last 4 frames and the first one
        dict(name="window-video-16384", kind="window", queries=16384, keys=16384, p0=0, heads=32, kv_heads=32, window=4,
             sinks=1024, frame=1024),
        # a decode step of 32 sequences: one token each
        dict(name="append-32x1", kind="append", seqs=32, rows=1, keys=4000, heads=32, kv_heads=8, page=16, layout=1),
        # the prompts of 9 requests, ragged
        dict(name="append-9-prompts", kind="append", seqs=9, rows=1777, keys=1777, heads=32, kv_heads=8, page=64, layout=2),
        # one user's next token
        dict(name="attend-1x1", kind="attend", seqs=1, rows=1, keys=1900, heads=32, kv_heads=8, page=16, tree=0, window=0,
             sinks=0, layout=3),
        # a decode step of 64 sequences, one query head for each key head
        dict(name="attend-64x1", kind="attend", seqs=64, rows=1, keys=7000, heads=16, kv_heads=16, page=64, tree=0, window=0,
             sinks=0, layout=5),
        # drafted trees of up to 64 tokens over long contexts, grouped heads
        dict(name="attend-tree-16x64", kind="attend", seqs=16, rows=64, keys=30000, heads=64, kv_heads=8, page=32, tree=1,
             window=0, sinks=0, layout=6),
        # a request forked into two: its last, partly filled page copied in each of 32 layers
        dict(name="copy-1-page", kind="copy", layers=32, pages=1, pool=65, kv_heads=8, page=16, layout=7),
        # a pool compacted: 1,000 pages moved down in each of 16 layers
        dict(name="copy-1000-pages", kind="copy", layers=16, pages=1000, pool=2000, kv_heads=8, page=16, layout=8),
        # one user's accepted branch moved behind the context
        dict(name="move-1x4", kind="move", layers=32, seqs=1, rows=4, drafted=26, keys=777, kv_heads=8, page=16, layout=4),
        # the accepted branches of 40 sequences' trees moved behind their contexts, in each of 32 layers
        dict(name="move-40x5", kind="move", layers=32, seqs=40, rows=5, drafted=26, keys=200, kv_heads=8, page=16, layout=9),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    layout = rng.randrange(10, 1 << 30)
    kv = rng.choice([1, 2, 4, 8, 16])
    kind = rng.choice(["window", "window", "window", "append", "append", "attend", "attend", "attend", "copy", "move"])
    if kind == "window":
        heads = kv * rng.choice([1, 2, 3, 4])
        q = _log_int(rng, 1, 9000)
        keys = q + _log_int(rng, 1, 6000)
        if rng.random() < 0.5:
            frame, window, sinks = 1, _log_int(rng, 1, 4000), rng.choice([0, 1, 4, 65])
        else:
            frame, window, sinks = _log_int(rng, 60, 1600), rng.randrange(1, 6), rng.choice([0, 77, 512])
        while q * heads * max(keys // 3, window * frame + sinks) > 2 * 10 ** 9:
            kv, heads = max(1, kv // 2), max(1, kv // 2) * (heads // kv)
        # some of them over the rows that are there so far, some with rows left behind the last query's position
        return dict(kind=kind, queries=q, keys=keys, p0=keys - q - rng.randrange(0, min(40, keys - q + 1)), heads=heads,
                    kv_heads=kv, window=window, sinks=sinks, frame=frame)
    page = rng.choice([8, 16, 32, 64, 128])
    if kind == "append":
        rows = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 64, 1500)])
        seqs, heads = _log_int(rng, 1, 64 if rows <= 64 else 10), min(64, kv * rng.choice([1, 2, 4, 7, 8])) // kv * kv
        while seqs > 1 and seqs * rows * (heads + 2 * kv) > 450000:
            seqs //= 2
        return dict(kind=kind, seqs=seqs, rows=rows, keys=rows + _log_int(rng, 1, 3001), heads=heads, kv_heads=kv, page=page,
                    layout=layout)
    if kind == "attend":
        rows = rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 2, 64), _log_int(rng, 64, 200)])
        seqs = _log_int(rng, 1, 64)
        keys = rows + _log_int(rng, 8, 30000)
        heads = min(64, kv * rng.choice([1, 2, 4, 7, 8])) // kv * kv
        while seqs > 1 and (seqs * keys * rows * heads > 1800000000 or seqs * keys * kv > 6000000):
            seqs //= 2
        window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
        return dict(kind=kind, seqs=seqs, rows=rows, keys=keys, heads=heads, kv_heads=kv, page=page,
                    tree=int(rows > 1 and rng.random() < 0.6), window=window, sinks=rng.choice([0, 4]) if window else 0,
                    layout=layout)
    layers = rng.randrange(1, 33)
    if kind == "copy":
        n = _log_int(rng, 1, max(1, 1900000 // (layers * page * kv)))
        return dict(kind=kind, layers=layers, pages=n, pool=2 * n + rng.randrange(1, 9), kv_heads=kv, page=page, layout=layout)
    drafted = rng.randrange(8, 65)
    return dict(kind=kind, layers=layers, seqs=_log_int(rng, 1, 64), rows=rng.randrange(1, 9), drafted=drafted,
                keys=drafted + rng.randrange(10, 300), kv_heads=kv, page=page, layout=layout)


# ---------------------------------------------------------------------------------------------------- layouts
# What a serving loop's host side knows of a batch (lengths, page tables, trees), from the case's `layout` alone.
def _layout(case):
    rng = random.Random(case["layout"])
    B, rows, keys, ps = case["seqs"], case["rows"], case["keys"], case["page"]
    new, lens = [], []
    for b in range(B):
        n = rows if b == 0 or rows == 1 or case["kind"] == "move" else rng.randrange(max(1, rows // 2), rows + 1)
        least = max(n, keys // 2, case.get("drafted", 0) + n)
        top = keys if b == 0 else rng.randrange(least, keys + 1)
        new.append(n)
        lens.append(top)
    width = (keys + ps - 1) // ps
    need = sum((x + ps - 1) // ps for x in lens)
    pool = need + 3
    ids = list(range(pool))
    rng.shuffle(ids)
    table, at = [], 0
    for x in lens:
        k = (x + ps - 1) // ps
        table.append(ids[at:at + k] + [0] * (width - k))
        at += k
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(new=new, lens=lens, table=table, starts=starts, pool=pool, width=width, rng=rng)


def _trees(lay):
    """Parent-first trees: each drafted token's ancestors and itself, as sets of indices."""
    rng, out = random.Random(lay["starts"][-1] * 7 + 1), []
    for n in lay["new"]:
        sets = []
        for i in range(n):
            parent = rng.randrange(-1, i) if i and rng.random() < 0.7 else i - 1
            sets.append({i} | (sets[parent] if parent >= 0 else set()))
        out.append(sets)
    return out


def _words(sets, words):
    rows = []
    for s in sets:
        w = [0] * words
        for x in s:
            w[x >> 6] |= 1 << (x & 63)
        rows.append([x - (1 << 64) if x >= 1 << 63 else x for x in w])
    return rows


# ---------------------------------------------------------------------------------------------------- inputs
def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(BF16)


def _angles(n):
    """cos / sin rows [n, 64] of a one-dimensional rotation, angles in 64 bits."""
    inv = THETA ** (-torch.arange(64, dtype=torch.float64, device="cuda") / 64)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    s = dict(case=case)
    if kind == "window":
        W, N, H, HK = case["queries"], case["keys"], case["heads"], case["kv_heads"]
        s.update(q=_normal(g, W, H, D), k=_normal(g, N, HK, D), v=_normal(g, N, HK, D),
                 out=torch.empty(W, H, D, dtype=BF16, device="cuda"))
        return s
    HK, ps = case["kv_heads"], case["page"]
    if kind == "copy":
        rng = random.Random(case["layout"])
        ids = list(range(case["pool"]))
        rng.shuffle(ids)
        n = case["pages"]
        s.update(k=_normal(g, case["layers"], case["pool"], ps, HK, D), v=_normal(g, case["layers"], case["pool"], ps, HK, D),
                 src=_ints(ids[:n]), dst=_ints(ids[n:2 * n]))
        return s
    lay = _layout(case)
    s.update(starts=_ints(lay["starts"]), lens=_ints(lay["lens"]), table=_ints(lay["table"]))
    if kind == "move":
        # drafted tokens start behind the context at the sequence's last `drafted` positions; the accepted ones go to the
        # positions in front of them
        rng, src, dst = lay["rng"], [], []
        for L in lay["lens"]:
            c, r = L - case["drafted"], case["rows"]
            src += sorted(rng.sample(range(c, L), r))
            dst += list(range(c - r, c))
        s.update(k=_normal(g, case["layers"], lay["pool"], ps, HK, D), v=_normal(g, case["layers"], lay["pool"], ps, HK, D),
                 src=_ints(src), dst=_ints(dst))
        return s
    H, T = case["heads"], lay["starts"][-1]
    s.update(kp=_normal(g, lay["pool"], ps, HK, D), vp=_normal(g, lay["pool"], ps, HK, D),
             out=torch.empty(T, H, D, dtype=BF16, device="cuda"))
    if kind == "append":
        qkv = _normal(g, T, H + 2 * HK, D)   # the packed projection's rows
        s.update(q=qkv[:, :H], k=qkv[:, H:H + HK], v=qkv[:, H + HK:], tab=_angles(case["keys"]),
                 qw=torch.rand(D, generator=g, device="cuda") + 0.5, kw=torch.rand(D, generator=g, device="cuda") + 0.5)
        return s
    s.update(q=_normal(g, T, H, D), tree=None)
    if case["tree"]:
        words = (case["rows"] + 63) // 64
        s["tree"] = torch.tensor([w for sets in _trees(lay) for w in _words(sets, words)], dtype=torch.int64, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        from localrouter_amd import cache, ops
        if kind == "window":
            return ops.attention_window(s["q"], s["k"], s["v"], s["out"], window=c["window"], sinks=c["sinks"],
                                        frame=c["frame"], p0=c["p0"])
        if kind == "append":
            cache.append(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["table"], s["starts"], s["lens"], s["out"],
                         q_norm=s["qw"], k_norm=s["kw"], table=s["tab"], eps=EPS)
            return s["out"], s["kp"], s["vp"]
        if kind == "attend":
            return cache.attention(s["q"], s["kp"], s["vp"], s["table"], s["starts"], s["lens"], s["out"],
                                   max_rows=c["rows"], max_keys=c["keys"], tree=s["tree"], window=c["window"],
                                   sinks=c["sinks"])
        if kind == "copy":
            cache.copy_pages(s["k"], s["v"], s["src"], s["dst"])
        else:
            cache.move_rows(s["k"], s["v"], s["table"], s["starts"], s["src"], s["dst"], max_rows=c["rows"])
        return s["k"], s["v"]
    return {"window": _plain_window, "append": _plain_append, "attend": _plain_attend, "copy": _plain_copy,
            "move": _plain_move}[kind](s, c)


def _plain_softmax(s, seen, v):
    """softmax over the last dim of the scores s where seen, times v; rows that see nothing: 0."""
    s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = s.sum(-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(s, v) / total, 0.0)


def _plain_window(s, c):
    W, N, H, HK, fr = c["queries"], c["keys"], c["heads"], c["kv_heads"], c["frame"]
    q = s["q"].float().view(W, HK, H // HK, D).permute(1, 2, 0, 3).contiguous()
    k = s["k"].float().permute(1, 2, 0).contiguous()[:, None]
    v = s["v"].float().transpose(0, 1).contiguous()[:, None]
    j = torch.arange(N, device="cuda")
    f = (c["p0"] + torch.arange(W, device="cuda"))[:, None] // fr
    seen = (j // fr <= f) & ((j // fr > f - c["window"]) | (j < c["sinks"]))
    sc = torch.matmul(q, k).mul_(SCALE)
    o = _plain_softmax(sc, seen, v)
    return o.permute(2, 0, 1, 3).reshape(W, H, D).to(BF16)


def _token_slots(s, T):
    """Each token's sequence, index in it and slot."""
    t = torch.arange(T, device="cuda")
    b = (t[:, None] >= s["starts"][None, 1:]).sum(1)
    i = t - s["starts"][b]
    n = s["starts"][b + 1] - s["starts"][b]
    return b, i, s["lens"][b] - n + i


def _plain_append(s, c):
    b, _, slot = _token_slots(s, s["q"].shape[0])
    cos, sin = s["tab"][0][slot][:, None], s["tab"][1][slot][:, None]

    def turned(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, e = x[..., 0::2], x[..., 1::2]
        return torch.stack([cos * a - sin * e, sin * a + cos * e], -1).flatten(-2).to(BF16)

    page, row = s["table"][b, slot // c["page"]].long(), slot % c["page"]
    s["kp"][page, row] = turned(s["k"], s["kw"])
    s["vp"][page, row] = s["v"]
    return turned(s["q"], s["qw"]), s["kp"], s["vp"]


def _plain_attend(s, c):
    T, H, HK, R, N = s["q"].shape[0], c["heads"], c["kv_heads"], c["rows"], c["keys"]
    G, B = H // HK, c["seqs"]
    j = torch.arange(N, device="cuda")
    page, row = s["table"][:, j // c["page"]].long(), j % c["page"]
    k = s["kp"][page, row].float().permute(0, 2, 3, 1).contiguous()     # [B, HK, D, N]
    v = s["vp"][page, row].float().transpose(1, 2).contiguous()         # [B, HK, N, D]
    n = s["starts"][1:] - s["starts"][:-1]
    ctx = (s["lens"] - n)[:, None]
    i = torch.arange(R, device="cuda")
    tok = (s["starts"][:-1, None] + i).clamp(max=T - 1)
    q = s["q"].float()[tok].view(B, R, HK, G, D).permute(0, 2, 3, 1, 4).reshape(B, HK, G * R, D)
    pos = ctx + i
    if c["tree"]:
        x = (j - ctx).clamp(0, 64 * s["tree"].shape[1] - 1)             # [B, N] drafted index of a key
        word = s["tree"][tok].gather(2, (x // 64)[:, None].expand(B, R, N))
        seen = (((word >> (x % 64)[:, None]) & 1) != 0) & (j < s["lens"][:, None])[:, None]
        bit = torch.arange(R, device="cuda")
        pos = ctx + ((s["tree"][tok][:, :, bit // 64] >> (bit % 64)) & 1).sum(-1) - 1
        seen |= j < ctx[:, None]
    else:
        seen = j <= pos[:, :, None]
    if c["window"]:
        far = (pos[:, :, None] - j >= c["window"]) & (j >= c["sinks"])
        seen &= ~(far & (j < ctx[:, None])) if c["tree"] else ~far
    sc = torch.matmul(q, k).mul_(SCALE).view(B, HK, G, R, N)
    o = _plain_softmax(sc, seen[:, None, None], v[:, :, None])          # [B, HK, G, R, D]
    b, i, _ = _token_slots(s, T)
    return o.permute(0, 3, 1, 2, 4).reshape(B, R, H, D)[b, i].to(BF16)


def _plain_copy(s, c):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return s["k"], s["v"]


def _plain_move(s, c):
    m = torch.arange(s["src"].shape[0], device="cuda")
    b = (m[:, None] >= s["starts"][None, 1:]).sum(1)
    ps = c["page"]
    sp, dp = s["table"][b, s["src"] // ps].long(), s["table"][b, s["dst"] // ps].long()
    s["k"][:, dp, s["dst"] % ps] = s["k"][:, sp, s["src"] % ps]
    s["v"][:, dp, s["dst"] % ps] = s["v"][:, sp, s["src"] % ps]
    return s["k"], s["v"]


# ---------------------------------------------------------------------------------------------------- work
def _window_range(c, i):
    """[lo, hi) and the sinks' end of the keys that query i sees."""
    f = (c["p0"] + i) // c["frame"]
    hi = min(c["keys"], (f + 1) * c["frame"])
    lo = min(max(0, (f - c["window"] + 1) * c["frame"]), hi)
    return lo, hi, min(c["sinks"], lo)


def work(case):
    c, kind = case, case["kind"]
    row = 2 * D
    if kind == "window":
        pairs = 0
        for i in range(c["queries"]):
            lo, hi, sk = _window_range(c, i)
            pairs += hi - lo + sk
        first, last = _window_range(c, 0), _window_range(c, c["queries"] - 1)
        keys = last[1] - first[0] + min(c["sinks"], first[0])
        return dict(bytes=2 * c["queries"] * c["heads"] * row + 2 * keys * c["kv_heads"] * row,
                    flops=4 * D * c["heads"] * pairs)
    if kind == "copy":
        return dict(bytes=4 * c["layers"] * c["pages"] * c["page"] * c["kv_heads"] * row, flops=0)
    if kind == "move":
        return dict(bytes=4 * c["layers"] * c["seqs"] * c["rows"] * c["kv_heads"] * row, flops=0)
    lay = _layout(c)
    T = lay["starts"][-1]
    if kind == "append":
        return dict(bytes=2 * T * (c["heads"] + 2 * c["kv_heads"]) * row + 512 * min(T, c["keys"]),
                    flops=8 * T * (c["heads"] + c["kv_heads"]) * D)
    trees = _trees(lay) if c["tree"] else None
    pairs = keys = 0
    for b, (n, L) in enumerate(zip(lay["new"], lay["lens"])):
        ctx, first = L - n, L
        for i in range(n):
            drafted = len(trees[b][i]) if trees else i + 1
            lo = max(0, ctx + drafted - c["window"]) if c["window"] else 0
            if trees:
                pairs += max(0, ctx - lo) + min(c["sinks"], lo, ctx) + drafted
            else:
                pairs += ctx + i + 1 - lo + min(c["sinks"], lo)
            first = min(first, lo, ctx if trees else lo)
        keys += L - first + min(c["sinks"], first)
    return dict(bytes=2 * keys * c["kv_heads"] * row + 2 * T * c["heads"] * row, flops=4 * D * c["heads"] * pairs)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"window": _exact_window, "append": _exact_append, "attend": _exact_attend, "copy": _exact_copy,
            "move": _exact_move}[case["kind"]](s, case)


def _exact_rows(q, k, v, hidden):
    """q [n, H, D] over k, v [m, HK, D] in 64 bits; hidden [n, m]: pairs left out (None: none)."""
    H, HK = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for h in range(H):
        kh, vh = k[:, h * HK // H].double(), v[:, h * HK // H].double()
        a = (q[:, h].double() @ kh.t().contiguous()) / math.sqrt(D)
        if hidden is not None:
            a[hidden] = -math.inf
        some = (a > -math.inf).any(1)
        out[some, h] = torch.softmax(a[some], 1) @ vh
    return out


def _exact_window(s, c):
    W = c["queries"]
    out = torch.empty(W, c["heads"], D, dtype=torch.float64, device="cuda")
    step = max(256, -(-W // 40))
    for i0 in range(0, W, step):
        i1 = min(W, i0 + step)
        spans = [_window_range(c, i) for i in range(i0, i1)]
        at = list(range(min(x[0] for x in spans), max(x[1] for x in spans)))
        at = list(range(0, min(c["sinks"], at[0] if at else 0))) + at
        j = torch.tensor(at, device="cuda")
        lo, hi, _ = (torch.tensor(x, device="cuda")[:, None] for x in zip(*spans))
        hidden = (j >= hi) | ((j < lo) & (j >= c["sinks"]))
        out[i0:i1] = _exact_rows(s["q"][i0:i1], s["k"][j], s["v"][j], hidden)
    return out


def _exact_append(s, c):
    lay = _layout(c)
    q, kp, vp = s["q"].double(), s["kp"].double(), s["vp"].double()
    for b, (n, L) in enumerate(zip(lay["new"], lay["lens"])):
        t0 = lay["starts"][b]
        z = torch.complex(s["tab"][0][L - n:L].double(), s["tab"][1][L - n:L].double())[:, None]

        def turned(x, w):
            x = x.double()
            x = x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], D // 2, 2)) * z).reshape(x.shape)

        k, q[t0:t0 + n] = turned(s["k"][t0:t0 + n], s["kw"]), turned(s["q"][t0:t0 + n], s["qw"])
        at = 0
        while at < n:   # one page's rows at a time
            p, r = divmod(L - n + at, c["page"])
            m = min(n - at, c["page"] - r)
            kp[lay["table"][b][p], r:r + m] = k[at:at + m]
            vp[lay["table"][b][p], r:r + m] = s["v"][t0 + at:t0 + at + m].double()
            at += m
    return q, kp, vp


def _exact_attend(s, c):
    lay = _layout(c)
    if c["heads"] * sum(n * L for n, L in zip(lay["new"], lay["lens"])) > 3e9:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    trees = _trees(lay) if c["tree"] else None
    for b, (n, L) in enumerate(zip(lay["new"], lay["lens"])):
        ctx, t0 = L - n, lay["starts"][b]
        pages = s["table"][b, :(L + c["page"] - 1) // c["page"]].long()
        k, v = (x[pages].flatten(0, 1)[:L] for x in (s["kp"], s["vp"]))
        hidden = torch.zeros(n, L, dtype=torch.bool)
        for i in range(n):
            if trees:
                hidden[i, ctx:] = True
                hidden[i, [ctx + x for x in trees[b][i]]] = False
                p = ctx + len(trees[b][i]) - 1
            else:
                hidden[i, ctx + i + 1:] = True
                p = ctx + i
            if c["window"]:
                edge = min(p - c["window"] + 1, ctx) if trees else p - c["window"] + 1
                if edge > c["sinks"]:
                    hidden[i, c["sinks"]:edge] = True
        out[t0:t0 + n] = _exact_rows(s["q"][t0:t0 + n], k, v, hidden.cuda())
    return out


def _exact_copy(s, c):
    src, dst = s["src"].tolist(), s["dst"].tolist()
    k, v = s["k"].clone(), s["v"].clone()
    for a, b in zip(src, dst):
        k[:, b].copy_(s["k"][:, a])
        v[:, b].copy_(s["v"][:, a])
    return k, v


def _exact_move(s, c):
    table, starts, ps = s["table"].tolist(), s["starts"].tolist(), c["page"]
    src, dst = s["src"].tolist(), s["dst"].tolist()
    k, v = s["k"].clone(), s["v"].clone()
    for b in range(c["seqs"]):
        for a, e in zip(src[starts[b]:starts[b + 1]], dst[starts[b]:starts[b + 1]]):
            for x, y in ((k, s["k"]), (v, s["v"])):
                x[:, table[b][e // ps], e % ps].copy_(y[:, table[b][a // ps], a % ps])
    return k, v
