"""ctypes mirror of include/lr_cache.h for torch tensors: a key / value cache in pages.

    append(q, k, v, k_pages, v_pages, page_table, starts, lens, ...)   norms, rotation and the write of new tokens, one pass
    attention(q, k_pages, v_pages, page_table, starts, lens, ...)      decode steps, chunks, drafted trees, windows
    copy_pages(k_pages, v_pages, src, dst)                             pages copied inside the pool, in every layer
    move_rows(k_pages, v_pages, page_table, starts, src, dst, ...)     rows moved inside their sequences, in every layer
    PagePool(n_pages)                                                  which pages are free, and who shares one (host only)

k_pages / v_pages: bf16 [n_pages, page_size, heads, 128] (copy_pages and move_rows also [layers, ...]), the same strides in
both; a pool laid out head by head is the permuted view of [n_pages, heads, page_size, 128]. page_table: int32 [B, pages a
sequence]; starts: int32 [B + 1], the call's tokens of sequence b being rows starts[b] .. starts[b + 1]; lens: int32 [B], the
sequences' lengths with those tokens. All on the current device.

Every call validates shapes on the host, then goes through the C ABI on torch's current HIP stream. There is no fallback:
without the built library every call raises.
"""
from __future__ import annotations

import ctypes
from pathlib import Path

import torch

from . import _lib
from .ops import D, PAIR_INTERLEAVED, SCALE_128, TABLE_COSSIN_F32, TABLE_NONE, _ptr, _rows, _stream

HEADER = Path(__file__).resolve().parent.parent / "include" / "lr_cache.h"

_P, _I, _I64, _F, _SZ = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t

SIGNATURES = {
    "lr_cache_append_bf16": (_I, [_P, _P, _P, _I64, _I64, _I64, _P, _I64, _P, _P, _I64, _I64, _I64, _I, _I, _P, _I64, _I, _P,
                                  _P, _P, _I, _I, _I, _I, _P, _P, _I, _P, _P, _I64, _I, _I, _I, _F, _P]),
    "lr_cache_attention_ws_bytes": (_SZ, [_I] * 9),
    "lr_cache_attention_bf16": (_I, [_P, _I64, _P, _I64, _P, _P, _I64, _I64, _I64, _I, _I, _P, _I64, _I, _P, _P, _I, _I, _I,
                                     _I, _I, _I, _P, _I, _I, _I, _F, _P, _SZ, _P]),
    "lr_cache_copy_pages": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I, _I, _I, _P, _P, _I, _P]),
    "lr_cache_move_rows": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I, _I, _I, _P, _I64, _I, _P, _P, _P, _I, _I, _I, _P]),
}

_bound = None


def lib() -> ctypes.CDLL:
    global _bound
    if _bound is None:
        L = _lib.load()
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _bound = L
    return _bound


def _call(name: str, *args) -> None:
    rc = getattr(lib(), name)(*args)
    if rc != 0:
        raise _lib.LrError(name, rc)


def _here(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda or t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"{name}: expected a tensor on the current device, got {t.device}")


def _ints(t: torch.Tensor, name: str, n: int) -> int:
    _here(t, name)
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] < n or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name}: expected contiguous int32 [{n}], got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _pool(k: torch.Tensor, v: torch.Tensor, layers: bool = False):
    """(k pointer, v pointer, [layers, layer stride,] page, row and head strides, pages, page size, heads)."""
    for t, name in ((k, "k_pages"), (v, "v_pages")):
        _here(t, name)
        if t.dtype != torch.bfloat16 or t.shape[-1] != D or t.stride(-1) != 1:
            raise ValueError(f"{name}: expected bf16 rows of 128 with unit stride, got {t.dtype} {tuple(t.shape)}")
    s, st = k.shape, k.stride()
    if v.shape != s or v.stride() != st:
        raise ValueError("k_pages and v_pages need the same shape and strides")
    if len(s) == 4:
        lead = (1, 0) if layers else ()
    elif len(s) == 5 and layers:
        lead = (s[0], st[0] if s[0] > 1 else 0)
    else:
        raise ValueError(f"k_pages: expected [n_pages, page_size, heads, 128]{' or [layers, ...]' if layers else ''}, got {tuple(s)}")
    P, R, H = s[-4:-1]
    # (a dimension of one element has whatever stride its view left: taken as packed)
    hs = st[-2] if H > 1 else D
    rs = st[-3] if R > 1 else max(D, (H - 1) * hs + D)
    ps = st[-4] if P > 1 else max((R - 1) * rs, 0) + (H - 1) * hs + D
    return (k.data_ptr(), v.data_ptr(), *lead, ps, rs, hs, P, R, H)


def _table(t: torch.Tensor, B: int):
    _here(t, "page_table")
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] < B or t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"page_table: expected int32 [{B}, pages] with contiguous rows, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else t.shape[1], t.shape[1]


def append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
           page_table: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, q_out: torch.Tensor | None = None, *,
           q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, table_kind: int = TABLE_COSSIN_F32,
           table: tuple | None = None, positions: torch.Tensor | None = None, pairing: int = PAIR_INTERLEAVED, rot: int = 128,
           eps: float = 1e-6) -> torch.Tensor | None:
    """lr_cache_append_bf16: new tokens q [T, H, 128], k / v [T, HK, 128] (views of a packed projection allowed): queries
    normalised and rotated into q_out (allocated when None; q itself is allowed), keys the same way into their pages, values
    as they are. table = (table_a, table_b), one row a position; positions int32 [T]: each token's table row (default its
    position in its sequence). q None: keys and values only. Returns q_out."""
    T, HK = k.shape[0], k.shape[1]
    B = lens.shape[0]
    H, q_rs, o_rs = 0, 0, 0
    k_rs, v_rs = _rows(k, "k", HK), _rows(v, "v", HK)
    _here(k, "k")
    _here(v, "v")
    if v.shape[0] != T:
        raise ValueError("append: k and v of different lengths")
    if q is not None:
        H = q.shape[1]
        q_rs = _rows(q, "q", H)
        _here(q, "q")
        if q.shape[0] != T:
            raise ValueError("append: q and k of different lengths")
        if q_out is None:
            q_out = torch.empty((T, H, D), dtype=torch.bfloat16, device=q.device)
        o_rs = _rows(q_out, "q_out", H)
        _here(q_out, "q_out")
        if q_out.shape[0] < T:
            raise ValueError("append: q_out shorter than q")
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _here(t, name)
            if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != D:
                raise ValueError(f"{name}: expected fp32 [128]")
    ta = tb = None
    stride = rows = 0
    if table_kind != TABLE_NONE:
        if table is None:
            raise ValueError("append: table required")
        ta, tb = table
        stride, rows = ta.stride(0), ta.shape[0]
        want = torch.bfloat16 if table_kind == 2 else torch.float32
        for t in (ta,) if tb is None else (ta, tb):
            _here(t, "table")
            if t.dtype != want or t.stride(0) != stride or t.shape[0] != rows:
                raise ValueError(f"table: expected {want} tensors of the same rows and row stride")
    pool = _pool(k_pages, v_pages)
    if pool[-1] != HK:
        raise ValueError(f"append: {HK} key heads, the pool has {pool[-1]}")
    _call("lr_cache_append_bf16", _ptr(q), k.data_ptr(), v.data_ptr(), q_rs, k_rs, v_rs, _ptr(q_out) if q is not None else None,
          o_rs, *pool[:7], *_table(page_table, B), _ints(starts, "starts", B + 1), _ints(lens, "lens", B),
          None if positions is None else _ints(positions, "positions", T), B, T, H, HK, _ptr(q_norm), _ptr(k_norm), table_kind,
          _ptr(ta), _ptr(tb), stride, rows, pairing, rot, eps, _stream())
    return q_out


def attention_ws_bytes(B: int, T: int, max_rows: int, max_keys: int, heads: int, kv_heads: int, page_size: int, *,
                       window: int = 0, sinks: int = 0) -> int:
    """lr_cache_attention_ws_bytes: the workspace a call needs (0: none)."""
    return int(lib().lr_cache_attention_ws_bytes(B, T, max_rows, max_keys, heads, kv_heads, page_size, window, sinks))


def attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
              lens: torch.Tensor, out: torch.Tensor | None = None, *, max_rows: int | None = None,
              max_keys: int | None = None, tree: torch.Tensor | None = None, window: int = 0, sinks: int = 0,
              scale: float = SCALE_128, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """lr_cache_attention_bf16: the batch's tokens q [T, H, 128] over their sequences' pages (append first). The token at
    position p sees positions j <= p; with tree (int64 [T, words], bit x of a token's words: it sees the sequence's x-th token
    of the call) drafted tokens see everything before the call's tokens and what their bits say. window n >= 1: earlier
    positions (under a tree: those before the call's tokens) only where p - j < n or j < sinks. max_rows: the most tokens of a
    sequence (default T); max_keys: the longest sequence (default what the table holds). A workspace of attention_ws_bytes is
    allocated when none is given."""
    T, H = q.shape[0], q.shape[1]
    B = lens.shape[0]
    q_rs = _rows(q, "q", H)
    _here(q, "q")
    pool = _pool(k_pages, v_pages)
    ps, HK = pool[6], pool[7]
    if out is None:
        out = torch.empty((T, H, D), dtype=torch.bfloat16, device=q.device)
    o_rs = _rows(out, "out", H)
    _here(out, "out")
    if out.shape[0] < T:
        raise ValueError("attention: out shorter than q")
    tab = _table(page_table, B)
    max_rows = T if max_rows is None else min(max_rows, T)
    max_keys = tab[2] * ps if max_keys is None else min(max_keys, tab[2] * ps)
    words = 0
    if tree is not None:
        _here(tree, "tree")
        if tree.dtype != torch.int64 or tree.dim() != 2 or tree.shape[0] < T or not tree.is_contiguous():
            raise ValueError(f"tree: expected contiguous int64 [{T}, words], got {tree.dtype} {tuple(tree.shape)}")
        words = tree.shape[1]
    need = attention_ws_bytes(B, T, max_rows, max_keys, H, HK, ps, window=window, sinks=sinks)
    nbytes = 0
    if workspace is not None:
        _here(workspace, "workspace")
        nbytes = workspace.numel() * workspace.element_size()
        if nbytes < need or not workspace.is_contiguous():
            raise ValueError(f"workspace: {need} contiguous bytes needed")
    elif need:
        workspace, nbytes = torch.empty(need, dtype=torch.uint8, device=q.device), need
    _call("lr_cache_attention_bf16", q.data_ptr(), q_rs, out.data_ptr(), o_rs, *pool[:7], *tab, _ints(starts, "starts", B + 1),
          _ints(lens, "lens", B), B, T, max_rows, max_keys, H, HK, _ptr(tree), words, window, sinks, scale, _ptr(workspace),
          nbytes, _stream())
    return out


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """lr_cache_copy_pages: page src[i] to page dst[i] (int32 [n] on the device) in every layer of [layers, n_pages, page_size,
    heads, 128] (or one layer's pool). No target may occur twice or be a source."""
    n = src.shape[0]
    pool = _pool(k_pages, v_pages, layers=True)
    if dst.shape[0] != n:
        raise ValueError("copy_pages: src and dst of different lengths")
    if n:
        _call("lr_cache_copy_pages", *pool, _ints(src, "src", n), _ints(dst, "dst", n), n, _stream())


def move_rows(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
              src: torch.Tensor, dst: torch.Tensor, *, max_rows: int | None = None) -> None:
    """lr_cache_move_rows: for the moves starts[b] .. starts[b + 1] of sequence b, its position src[i] to its position dst[i],
    in every layer; a sequence's rows are all read before any is written. max_rows: the most moves of a sequence (at most 256;
    default all of them)."""
    n, B = src.shape[0], starts.shape[0] - 1
    pool = _pool(k_pages, v_pages, layers=True)
    if dst.shape[0] != n:
        raise ValueError("move_rows: src and dst of different lengths")
    if n:
        _call("lr_cache_move_rows", *pool, *_table(page_table, B), _ints(starts, "starts", B + 1), _ints(src, "src", n),
              _ints(dst, "dst", n), B, n, n if max_rows is None else min(max_rows, n), _stream())


class PagePool:
    """Which of a pool's pages are free and how many sequences hold each: host bookkeeping beside the calls above.

    alloc / fork / free change holders only. own() is for a sequence about to write into a page that others hold too: it gives
    the sequence a page of its own and says what to copy. compact() packs the used pages to the front of the pool. The pairs
    these return go to copy_pages."""

    def __init__(self, n_pages: int):
        if n_pages < 1:
            raise ValueError("PagePool: at least one page")
        self.holders = [0] * n_pages
        self._free = list(range(n_pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def alloc(self, n: int) -> list[int]:
        """n pages, held once; raises MemoryError, and takes none, when fewer are free."""
        if n < 0:
            raise ValueError("alloc: negative count")
        if n > len(self._free):
            raise MemoryError(f"PagePool: {n} pages asked for, {len(self._free)} free")
        pages = [self._free.pop() for _ in range(n)]
        for p in pages:
            self.holders[p] = 1
        return pages

    def _held(self, pages) -> None:
        for p in pages:
            if not 0 <= p < len(self.holders) or self.holders[p] == 0:
                raise ValueError(f"PagePool: page {p} is not held")

    def fork(self, pages: list[int]) -> list[int]:
        """The same pages for another sequence."""
        self._held(pages)
        for p in pages:
            self.holders[p] += 1
        return list(pages)

    def free(self, pages: list[int]) -> None:
        """One holder fewer for each page; a page without one is free again."""
        self._held(pages)
        if any(self.holders[p] < pages.count(p) for p in set(pages)):
            raise ValueError("PagePool: a page freed more often than it is held")
        for p in pages:
            self.holders[p] -= 1
            if self.holders[p] == 0:
                self._free.append(p)

    def own(self, pages: list[int], index: int) -> tuple[int, int] | None:
        """Makes pages[index] the sequence's own (in place): None when no one else holds it, else (source, target) to copy."""
        p = pages[index]
        self._held([p])
        if self.holders[p] == 1:
            return None
        q, = self.alloc(1)
        self.holders[p] -= 1
        pages[index] = q
        return p, q

    def compact(self, tables: list[list[int]]) -> tuple[list[int], list[int]]:
        """Moves the pages of `tables` (every holder's list, changed in place) to the front of the pool. Returns (sources,
        targets): the targets were free, so no page is both."""
        seen: dict[int, int] = {}
        for t in tables:
            for p in t:
                seen[p] = seen.get(p, 0) + 1
        self._held(seen)
        used = sum(h > 0 for h in self.holders)
        if len(seen) != used or any(self.holders[p] != n for p, n in seen.items()):
            raise ValueError("PagePool: compact needs the tables of every holder")
        holes = [p for p in range(used) if self.holders[p] == 0]
        src = sorted((p for p in seen if p >= used), reverse=True)
        to = dict(zip(src, holes))
        for a, b in to.items():
            self.holders[b], self.holders[a] = self.holders[a], 0
        for t in tables:
            t[:] = [to.get(p, p) for p in t]
        self._free = list(range(len(self.holders) - 1, used - 1, -1))
        return list(to), list(to.values())
