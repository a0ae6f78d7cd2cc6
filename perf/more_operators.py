"""The cache in 8-bit pages and attention over packed prompts, as cases that can be timed and compared.

  packed   ops.attention_packed: the tokens of B sequences end to end, sequence b the rows starts[b] .. starts[b + 1]; its token i
           sees its tokens j <= i, with a window of n those with i - j < n or j < sinks; out_i = softmax(scale * q_i k_j) v_j
  append   cache.append_f8: token t of sequence b takes slot s = lens[b] - n_b + (t - starts[b]) of its sequence (n_b of the tokens
           are sequence b's, lens[b] counts them); per head y = x / sqrt(mean(x^2) + eps) * w, pairs rotated by the table row of
           the token's position; q to bf16 rows, k and v to 8 bits: row s % page_size of page page_table[b][s // page_size]. 16
           rows of a page and head share a scale 2^e: the least e with max|y| <= 448 * 2^e over the sequence's new rows among them,
           and no less than before where earlier rows of the sequence lie among them, which are then rounded again to the new scale
  attend   cache.attention_f8: the tokens of each sequence over its pages, key j of head g being page row times scale. The token of
           slot p sees j <= p; drafted tokens under a tree see the context j < c = lens[b] - n_b and the drafted keys c + x whose
           bit x is set in the token's mask; with a window of n positions, context further back than that and not among the sinks
           is left out

  listed()             the named cases
  draw(rng)            one more case of the same ranges
  prepare(case, seed)  the inputs and what a program keeps between calls (pools, page tables, output buffers)
  run(state)           one pass; returns its outputs (8-bit pages and scales as the tensors they are: both are float types)
  work(case)           the bytes and floating-point operations the pass cannot do without
  exact(case, seed)    the outputs in 64 bits (of 8-bit pages the quotients that were rounded; of scales none)

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
GROUP = 16            # rows of a page that share a scale
TOP = 448.0           # the largest e4m3 value
BF16, F8, E8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # three short prompts of a chat's first turn: latency
        dict(name="packed-3-short", kind="packed", seqs=3, rows=41, heads=32, kv_heads=8, window=0, sinks=0, layout=1),
        # a batch of 19 requests' prompts, ragged, grouped heads
        dict(name="packed-19-prompts", kind="packed", seqs=19, rows=1100, heads=32, kv_heads=8, window=0, sinks=0, layout=2),
        # text encodings of 40 captions, a key head for each query head
        dict(name="packed-40-captions", kind="packed", seqs=40, rows=257, heads=16, kv_heads=16, window=0, sinks=0, layout=3),
        # documents of up to 7,000 tokens packed into one training-length batch
        dict(name="packed-4-documents", kind="packed", seqs=4, rows=7000, heads=32, kv_heads=4, window=0, sinks=0, layout=4),
        # a decode step of 24 sequences: one token each, most of them into a block that holds tokens already
        dict(name="append8-24x1", kind="append", seqs=24, rows=1, keys=700, heads=32, kv_heads=8, page=16, layout=5),
        # drafted tokens of 7 sequences, ragged, behind partly filled blocks
        dict(name="append8-7x37", kind="append", seqs=7, rows=37, keys=450, heads=64, kv_heads=8, page=32, layout=6),
        # the prompts of 11 requests, ragged
        dict(name="append8-11-prompts", kind="append", seqs=11, rows=1500, keys=1500, heads=32, kv_heads=8, page=64, layout=7),
        # one user's next token
        dict(name="attend8-1x1", kind="attend", seqs=1, rows=1, keys=2100, heads=32, kv_heads=8, page=16, tree=0, window=0, sinks=0,
             layout=8),
        # a decode step of 48 sequences of up to 9,000 positions
        dict(name="attend8-48x1", kind="attend", seqs=48, rows=1, keys=9000, heads=32, kv_heads=8, page=64, tree=0, window=0,
             sinks=0, layout=9),
        # drafted trees of up to 9 tokens over long contexts
        dict(name="attend8-tree-20x9", kind="attend", seqs=20, rows=9, keys=12000, heads=24, kv_heads=8, page=32, tree=1, window=0,
             sinks=0, layout=10),
        # chunks of 700 tokens of 2 prompts behind 5,000 positions
        dict(name="attend8-chunk-2x700", kind="attend", seqs=2, rows=700, keys=5700, heads=32, kv_heads=8, page=16, tree=0, window=0,
             sinks=0, layout=11),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    layout = rng.randrange(20, 1 << 30)
    kv = rng.choice([1, 2, 4, 8, 16])
    kind = rng.choice(["packed", "packed", "packed", "append", "append", "attend", "attend", "attend"])
    if kind == "packed":
        heads = min(64, kv * rng.choice([1, 2, 3, 4, 8])) // kv * kv
        seqs = _log_int(rng, 1, 60)
        rows = _log_int(rng, 1, 7000)
        while seqs > 1 and seqs * rows * rows * heads > 6 * 10 ** 9:
            seqs //= 2
        while heads > kv and rows * rows * heads > 6 * 10 ** 9:
            heads = kv
        window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
        return dict(kind=kind, seqs=seqs, rows=rows, heads=heads, kv_heads=kv, window=window,
                    sinks=rng.choice([0, 4, 65]) if window else 0, layout=layout)
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        rows = rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 64, 1500)])
        seqs, heads = _log_int(rng, 1, 64 if rows <= 64 else 10), min(64, kv * rng.choice([1, 2, 4, 7, 8])) // kv * kv
        while seqs > 1 and seqs * rows * (heads + 2 * kv) > 400000:
            seqs //= 2
        return dict(kind=kind, seqs=seqs, rows=rows, keys=rows + _log_int(rng, 1, 900), heads=heads, kv_heads=kv, page=page,
                    layout=layout)
    rows = rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 2, 64), _log_int(rng, 64, 700)])
    seqs = _log_int(rng, 1, 64)
    keys = rows + _log_int(rng, 8, 20000)
    heads = min(64, kv * rng.choice([1, 2, 4, 7, 8])) // kv * kv
    while seqs > 1 and (seqs * keys * rows * heads > 250 * 10 ** 6 or seqs * keys * kv > 3400000):
        seqs //= 2
    while keys > rows + 16 and keys * rows * heads > 250 * 10 ** 6:
        keys = rows + (keys - rows) // 2
    window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
    return dict(kind=kind, seqs=seqs, rows=rows, keys=keys, heads=heads, kv_heads=kv, page=page,
                tree=int(1 < rows <= 300 and rng.random() < 0.6), window=window, sinks=rng.choice([0, 4]) if window else 0,
                layout=layout)


# ---------------------------------------------------------------------------------------------------- layouts
# What a serving loop's host side knows of a batch (lengths, page tables, trees), from the case's `layout` alone.
def _lengths(case):
    """The packed sequences' lengths: the first has the most."""
    rng, n = random.Random(case["layout"]), case["rows"]
    return [n if b == 0 else rng.randrange(max(1, n // 20), n + 1) for b in range(case["seqs"])]


def _sums(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _layout(case):
    rng = random.Random(case["layout"])
    B, rows, keys, ps = case["seqs"], case["rows"], case["keys"], case["page"]
    new, lens = [], []
    for b in range(B):
        n = rows if b == 0 or rows == 1 else rng.randrange(max(1, rows // 2), rows + 1)
        new.append(n)
        lens.append(keys if b == 0 else rng.randrange(max(n, keys // 2), keys + 1))
    width = (keys + ps - 1) // ps
    held = [(x + ps - 1) // ps for x in lens]
    pool = sum(held) + 3
    ids = list(range(pool))
    rng.shuffle(ids)
    ends = _sums(held)
    table = [ids[ends[b]:ends[b + 1]] + [0] * (width - held[b]) for b in range(B)]
    return dict(new=new, lens=lens, table=table, starts=_sums(new), pool=pool)


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


def _exponent(a):
    """The least e with a <= 448 * 2^e, between -100 and 119."""
    m, x = torch.frexp(a)
    return torch.where(a > 0, torch.where(m > 0.875, x - 8, x - 9), -100).clamp(-100, 119)


def _pages(g, pool, ps, HK):
    """A pool as earlier calls left it: pages of normal values, heads of different magnitude, and their scales."""
    x = torch.randn((pool * ps // GROUP, GROUP, HK, D), generator=g, device="cuda")
    x *= torch.exp(torch.randn((HK, 1), generator=g, device="cuda"))
    e = _exponent(x.abs().amax((1, 3)))
    pages = torch.ldexp(x, -e[:, None, :, None]).to(F8).view(pool, ps, HK, D)
    return pages, (e + 127).to(torch.uint8).view(E8).view(pool, ps // GROUP, HK)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, H, HK = case["kind"], case["heads"], case["kv_heads"]
    s = dict(case=case)
    if kind == "packed":
        starts = _sums(_lengths(case))
        T = starts[-1]
        qkv = _normal(g, T, H + 2 * HK, D)   # the packed projection's rows
        s.update(q=qkv[:, :H], k=qkv[:, H:H + HK], v=qkv[:, H + HK:], starts=_ints(starts),
                 out=torch.empty(T, H, D, dtype=BF16, device="cuda"))
        return s
    lay = _layout(case)
    T = lay["starts"][-1]
    s.update(starts=_ints(lay["starts"]), lens=_ints(lay["lens"]), table=_ints(lay["table"]))
    s["kp"], s["ks"] = _pages(g, lay["pool"], case["page"], HK)
    s["vp"], s["vs"] = _pages(g, lay["pool"], case["page"], HK)
    s["out"] = torch.empty(T, H, D, dtype=BF16, device="cuda")
    if kind == "append":
        qkv = _normal(g, T, H + 2 * HK, D)
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
        if kind == "packed":
            return ops.attention_packed(s["q"], s["k"], s["v"], s["starts"], s["out"], window=c["window"], sinks=c["sinks"])
        if kind == "append":
            cache.append_f8(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["ks"], s["vs"], s["table"], s["starts"], s["lens"], s["out"],
                            q_norm=s["qw"], k_norm=s["kw"], table=s["tab"], eps=EPS)
            return s["out"], s["kp"], s["vp"], s["ks"], s["vs"]
        return cache.attention_f8(s["q"], s["kp"], s["vp"], s["ks"], s["vs"], s["table"], s["starts"], s["lens"], s["out"],
                                  max_rows=c["rows"], max_keys=c["keys"], tree=s["tree"], window=c["window"], sinks=c["sinks"])
    return {"packed": _plain_packed, "append": _plain_append, "attend": _plain_attend}[kind](s, c)


def _plain_softmax(s, seen, v):
    """softmax over the last dim of the scores s where seen, times v; rows that see nothing: 0."""
    s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = s.sum(-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(s, v) / total, 0.0)


def _plain_packed(s, c):
    # the sequences padded to the longest
    T, H, HK, R = s["q"].shape[0], c["heads"], c["kv_heads"], c["rows"]
    B, G = c["seqs"], H // HK
    i = torch.arange(R, device="cuda")
    at = (s["starts"][:-1, None] + i).clamp(max=T - 1)
    q = s["q"].float()[at].view(B, R, HK, G, D).permute(0, 2, 3, 1, 4).reshape(B, HK, G * R, D)
    k = s["k"].float()[at].permute(0, 2, 3, 1).contiguous()     # [B, HK, D, R]
    v = s["v"].float()[at].transpose(1, 2).contiguous()         # [B, HK, R, D]
    seen = i <= i[:, None]
    if c["window"]:
        seen &= (i > i[:, None] - c["window"]) | (i < c["sinks"])
    sc = torch.matmul(q, k).mul_(SCALE).view(B, HK, G, R, R)
    o = _plain_softmax(sc, seen, v[:, :, None]).permute(0, 3, 1, 2, 4).reshape(B, R, H, D)
    t = torch.arange(T, device="cuda")
    b = (t[:, None] >= s["starts"][None, 1:]).sum(1)
    return o[b, t - s["starts"][b]].to(BF16)


def _token_slots(s, T):
    """Each token's sequence, index in it and slot."""
    t = torch.arange(T, device="cuda")
    b = (t[:, None] >= s["starts"][None, 1:]).sum(1)
    i = t - s["starts"][b]
    n = s["starts"][b + 1] - s["starts"][b]
    return b, i, s["lens"][b] - n + i


def _exponents(scales):
    return scales.view(torch.uint8).flatten(0, 1).int() - 127


def _plain_store(x, pages, scales, page, row, leads):
    """fp32 rows x [T, HK, D] to rows `row` of `page`; leads: the first token of each sequence in each group of rows."""
    groups = pages.view(torch.uint8).view(-1, GROUP, x.shape[1], D)
    grp, r = page * (pages.shape[1] // GROUP) + row // GROUP, row % GROUP
    a = torch.zeros(len(groups), x.shape[1], device="cuda")
    a.scatter_reduce_(0, grp[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    e = _exponents(scales)
    at, first = grp[leads], r[leads]
    old = e[at]
    new = _exponent(a[at])
    new = torch.where(first[:, None] > 0, torch.maximum(new, old), new)
    bits = groups[at]
    again = torch.ldexp(bits.view(F8).float(), (old - new)[:, None, :, None]).to(F8).view(torch.uint8)
    groups[at] = torch.where((torch.arange(GROUP, device="cuda") < first[:, None])[:, :, None, None], again, bits)
    e[at] = new
    scales.view(torch.uint8).view(-1, x.shape[1])[at] = (new + 127).to(torch.uint8)
    groups[grp, r] = torch.ldexp(x, -e[grp][:, :, None]).clamp(-TOP, TOP).to(F8).view(torch.uint8)


def _plain_append(s, c):
    b, i, slot = _token_slots(s, s["q"].shape[0])
    cos, sin = s["tab"][0][slot][:, None], s["tab"][1][slot][:, None]

    def turned(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, e = x[..., 0::2], x[..., 1::2]
        return torch.stack([cos * a - sin * e, sin * a + cos * e], -1).flatten(-2)

    page, row = s["table"][b, slot // c["page"]].long(), slot % c["page"]
    leads = ((i == 0) | (slot % GROUP == 0)).nonzero()[:, 0]
    _plain_store(turned(s["k"], s["kw"]), s["kp"], s["ks"], page, row, leads)
    _plain_store(s["v"].float(), s["vp"], s["vs"], page, row, leads)
    return turned(s["q"], s["qw"]).to(BF16), s["kp"], s["vp"], s["ks"], s["vs"]


def _values(pages, scales):
    """The fp32 values of 8-bit pages [..., page_size, HK, D] and their scales [..., page_size / 16, HK]."""
    e = (scales.view(torch.uint8).int() - 127).repeat_interleave(GROUP, -2)
    return torch.ldexp(pages.float(), e[..., None])


def _plain_attend(s, c):
    T, H, HK, R, N = s["q"].shape[0], c["heads"], c["kv_heads"], c["rows"], c["keys"]
    G, B = H // HK, c["seqs"]
    j = torch.arange(N, device="cuda")
    page, row = s["table"][:, j // c["page"]].long(), j % c["page"]
    k = _values(s["kp"], s["ks"])[page, row].permute(0, 2, 3, 1).contiguous()     # [B, HK, D, N]
    v = _values(s["vp"], s["vs"])[page, row].transpose(1, 2).contiguous()         # [B, HK, N, D]
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
        seen &= ~(far & (j < ctx[:, None])[:, None]) if c["tree"] else ~far
    sc = torch.matmul(q, k).mul_(SCALE).view(B, HK, G, R, N)
    o = _plain_softmax(sc, seen[:, None, None], v[:, :, None])          # [B, HK, G, R, D]
    b, i, _ = _token_slots(s, T)
    return o.permute(0, 3, 1, 2, 4).reshape(B, R, H, D)[b, i].to(BF16)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    c, kind = case, case["kind"]
    row, H, HK = 2 * D, case["heads"], case["kv_heads"]
    if kind == "packed":
        lengths, T = _lengths(c), sum(_lengths(c))
        pairs = 0
        for n in lengths:
            w = min(c["window"], n) if c["window"] else n
            pairs += w * (w + 1) // 2 + (n - w) * w
            # first tokens that the window has left behind
            pairs += sum(min(c["sinks"], i + 1 - w) for i in range(w, n)) if c["sinks"] else 0
        return dict(bytes=2 * T * (H + HK) * row, flops=4 * D * H * pairs)
    lay = _layout(c)
    T = lay["starts"][-1]
    if kind == "append":
        return dict(bytes=T * (2 * H + 2 * HK) * row + T * HK * row + 512 * min(T, c["keys"]), flops=8 * T * (H + HK) * D)
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
    return dict(bytes=2 * keys * HK * D + keys * HK // 8 + 2 * T * H * row, flops=4 * D * H * pairs)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"packed": _exact_packed, "append": _exact_append, "attend": _exact_attend}[case["kind"]](s, case)


def _exact_rows(q, k, v, hidden):
    """q [n, H, D] over fp64 k, v [m, HK, D]; hidden [n, m]: pairs left out."""
    H, HK = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for h in range(H):
        a = (q[:, h].double() @ k[:, h * HK // H].t().contiguous()) / math.sqrt(D)
        a[hidden] = -math.inf
        some = (a > -math.inf).any(1)
        out[some, h] = torch.softmax(a[some], 1) @ v[:, h * HK // H]
    return out


def _exact_packed(s, c):
    starts = _sums(_lengths(c))
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for t0, t1 in zip(starts, starts[1:]):
        for i0 in range(0, t1 - t0, 2048):   # rows of a sequence, over the keys up to the last of them
            i1 = min(t1 - t0, i0 + 2048)
            back = torch.arange(i0, i1, device="cuda")[:, None] - torch.arange(i1, device="cuda")
            hidden = back < 0
            if c["window"]:
                hidden |= (back >= c["window"]) & (torch.arange(i1, device="cuda") >= c["sinks"])
            out[t0 + i0:t0 + i1] = _exact_rows(s["q"][t0 + i0:t0 + i1], s["k"][t0:t0 + i1].double(), s["v"][t0:t0 + i1].double(),
                                               hidden)
    return out


def _exact_append(s, c):
    lay = _layout(c)
    q = s["q"].double()
    pools = [s["kp"].double(), s["vp"].double()]
    for b, (n, L) in enumerate(zip(lay["new"], lay["lens"])):
        t0 = lay["starts"][b]
        z = torch.complex(s["tab"][0][L - n:L].double(), s["tab"][1][L - n:L].double())[:, None]

        def turned(x, w):
            x = x.double()
            x = x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], D // 2, 2)) * z).reshape(x.shape)

        q[t0:t0 + n] = turned(s["q"][t0:t0 + n], s["qw"])
        rows = [turned(s["k"][t0:t0 + n], s["kw"]), s["v"][t0:t0 + n].double()]
        at = 0
        while at < n:   # one group's rows at a time
            p, r = divmod(L - n + at, c["page"])
            page, grp, r0 = lay["table"][b][p], r // GROUP, r % GROUP
            m = min(n - at, GROUP - r0)
            for x, pool, scales in zip(rows, pools, (s["ks"], s["vs"])):
                y = x[at:at + m]
                e = torch.ceil(torch.log2(y.abs().amax((0, 2)) / TOP))                      # [HK]
                if r0:
                    old = scales[page, grp].view(torch.uint8).double() - 127
                    e = torch.maximum(e, old)
                    pool[page, r - r0:r] *= torch.exp2(old - e)[:, None]
                pool[page, r:r + m] = y * torch.exp2(-e)[:, None]
            at += m
    return q, pools[0], pools[1], None, None


def _exact_attend(s, c):
    lay = _layout(c)
    if c["heads"] * sum(n * L for n, L in zip(lay["new"], lay["lens"])) > 3e9:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    trees = _trees(lay) if c["tree"] else None
    for b, (n, L) in enumerate(zip(lay["new"], lay["lens"])):
        ctx, t0 = L - n, lay["starts"][b]
        pages = s["table"][b, :(L + c["page"] - 1) // c["page"]].long()
        k, v = ((p[pages].double().unflatten(1, (-1, GROUP)) * f.view(torch.uint8)[pages].double().sub(127).exp2()[:, :, None, :, None])
                .flatten(0, 2)[:L] for p, f in ((s["kp"], s["ks"]), (s["vp"], s["vs"])))
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
