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

import collections
import ctypes
import functools
from pathlib import Path

import torch

from . import _lib
from .ops import D, PAIR_INTERLEAVED, SCALE_128, TABLE_COSSIN_F32, TABLE_NONE

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

INT_MAX = 2 ** 31 - 1

_bound = None
_BF16, _I32, _I64T, _F32 = torch.bfloat16, torch.int32, torch.int64, torch.float32
# (looked up once: a small call's ~10 us are mostly its checks)
_current, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def lib() -> ctypes.CDLL:
    global _bound
    if _bound is None:
        L = _lib.load()
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _bound = L
    return _bound


def _device(t: torch.Tensor) -> int:
    """The current device; a host tensor is refused (there may be no device to ask)."""
    if not t.is_cuda:
        raise ValueError(f"expected tensors on the GPU, got one on {t.device}")
    return _current()


def _check(name: str, rc: int) -> None:
    if rc != 0:
        raise _lib.LrError(name, rc)


def _refuse(name: str, want: str, *tensors: torch.Tensor):
    got = ", ".join(f"{t.dtype} {tuple(t.shape)} / {tuple(t.stride())} on {t.device}" for t in tensors)
    raise ValueError(f"{name}: expected {want} on the current device, got {got}")


def _rows(t: torch.Tensor, name: str, dev: int, n: int, heads: int) -> int:
    """The row stride of bf16 rows [>= n, heads, 128] on device dev."""
    s, st = t.shape, t.stride()
    if (len(s) == 3 and s[0] >= n and s[1] == heads and s[2] == 128 and st[2] == 1 and (st[1] == 128 or heads == 1)
            and t.dtype is _BF16 and t.get_device() == dev):
        return st[0] if s[0] > 1 else heads * 128
    _refuse(name, f"bf16 [{n}, {heads}, 128] with contiguous heads", t)


def _ints(t: torch.Tensor, name: str, dev: int, n: int) -> int:
    s = t.shape
    if len(s) == 1 and s[0] >= n and t.dtype is _I32 and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    _refuse(name, f"contiguous int32 [{n}]", t)


def _pool(k: torch.Tensor, v: torch.Tensor, dev: int, layers: bool = False) -> tuple:
    """([layers, layer stride,] page, row and head strides, pages, page size, heads)."""
    s, st = k.shape, k.stride()
    n = len(s)
    if (v.shape != s or v.stride() != st or (n != 4 and (n != 5 or not layers)) or s[-1] != 128 or st[-1] != 1
            or k.dtype is not _BF16 or v.dtype is not _BF16 or k.get_device() != dev or v.get_device() != dev):
        _refuse("k_pages, v_pages", f"bf16 [n_pages, page_size, heads, 128]{' or [layers, ...]' if layers else ''} of the same "
                "shape and strides", k, v)
    if n == 4:
        P, R, H, _ = s
        ps, rs, hs, _ = st
    else:
        L, P, R, H, _ = s
        ls, ps, rs, hs, _ = st
    # (a dimension of one element has whatever stride its view left: taken as packed)
    if H == 1:
        hs = 128
    if R == 1:
        rs = (H - 1) * hs + 128
    if P == 1:
        ps = (R - 1) * rs + (H - 1) * hs + 128
    if layers:
        return (L, ls if L > 1 else 0, ps, rs, hs, P, R, H) if n == 5 else (1, 0, ps, rs, hs, P, R, H)
    return ps, rs, hs, P, R, H


def _table(t: torch.Tensor, dev: int, B: int) -> tuple:
    s, st = t.shape, t.stride()
    if len(s) == 2 and s[0] >= B and (st[1] == 1 or s[1] == 1) and t.dtype is _I32 and t.get_device() == dev:
        return t.data_ptr(), st[0] if s[0] > 1 else s[1], s[1]
    _refuse("page_table", f"int32 [{B}, pages] with contiguous rows", t)


def append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
           page_table: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, q_out: torch.Tensor | None = None, *,
           q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, table_kind: int = TABLE_COSSIN_F32,
           table: tuple | None = None, positions: torch.Tensor | None = None, pairing: int = PAIR_INTERLEAVED, rot: int = 128,
           eps: float = 1e-6) -> torch.Tensor | None:
    """lr_cache_append_bf16: new tokens q [T, H, 128], k / v [T, HK, 128] (views of a packed projection allowed): queries
    normalised and rotated into q_out (allocated when None; q itself is allowed), keys the same way into their pages, values
    as they are. table = (table_a, table_b), one row a position; positions int32 [T]: each token's table row (default its
    position in its sequence). q None: keys and values only. Returns q_out."""
    dev = _device(k_pages)
    ps, rs, hs, n_pages, page_size, HK = _pool(k_pages, v_pages, dev)
    T, B = k.shape[0], lens.shape[0]
    k_rs, v_rs = _rows(k, "k", dev, T, HK), _rows(v, "v", dev, T, HK)
    H = q_rs = o_rs = 0
    q_ptr = o_ptr = None
    if q is not None:
        H = q.shape[1]
        q_rs = _rows(q, "q", dev, T, H)
        if q_out is None:
            q_out = torch.empty((T, H, D), dtype=_BF16, device=q.device)
        o_rs = _rows(q_out, "q_out", dev, T, H)
        q_ptr, o_ptr = q.data_ptr(), q_out.data_ptr()
    if v.shape[0] != T or (q is not None and q.shape[0] != T):
        raise ValueError("append: q, k and v of different lengths")
    if T == 0:
        return q_out
    qw = kw = ta = tb = pos = None
    stride = rows = 0
    for t in (q_norm, k_norm):
        if t is not None and (t.dtype is not _F32 or t.numel() != 128 or not t.is_contiguous() or t.get_device() != dev):
            _refuse("q_norm, k_norm", "fp32 [128]", t)
    if q_norm is not None:
        qw = q_norm.data_ptr()
    if k_norm is not None:
        kw = k_norm.data_ptr()
    if table_kind != TABLE_NONE:
        if table is None:
            raise ValueError("append: table required")
        a, b = table
        want = _BF16 if table_kind == 2 else _F32
        st = a.stride()
        if a.dim() != 2 or st[1] != 1 or a.dtype is not want or a.get_device() != dev:
            _refuse("table", f"{want} rows", a)
        stride, rows, ta = st[0], a.shape[0], a.data_ptr()
        if b is not None:
            if b.shape != a.shape or b.stride() != st or b.dtype is not want or b.get_device() != dev:
                _refuse("table", "two tensors of the same type, shape and strides", a, b)
            tb = b.data_ptr()
    if positions is not None:
        pos = _ints(positions, "positions", dev, T)
    tab, tab_rs, tab_pages = _table(page_table, dev, B)
    _check("lr_cache_append_bf16", lib().lr_cache_append_bf16(
        q_ptr, k.data_ptr(), v.data_ptr(), q_rs, k_rs, v_rs, o_ptr, o_rs, k_pages.data_ptr(), v_pages.data_ptr(), ps, rs, hs,
        n_pages, page_size, tab, tab_rs, tab_pages, _ints(starts, "starts", dev, B + 1), _ints(lens, "lens", dev, B), pos, B, T,
        H, HK, qw, kw, table_kind, ta, tb, stride, rows, pairing, rot, eps, _raw_stream(dev)))
    return q_out


@functools.lru_cache(maxsize=1024)
def _ws_bytes(*sizes: int) -> int:
    return int(lib().lr_cache_attention_ws_bytes(*sizes))


def attention_ws_bytes(B: int, T: int, max_rows: int, max_keys: int, heads: int, kv_heads: int, page_size: int, *,
                       window: int = 0, sinks: int = 0) -> int:
    """lr_cache_attention_ws_bytes: the workspace a call needs (0: none)."""
    return _ws_bytes(B, T, max_rows, max_keys, heads, kv_heads, page_size, window, sinks)


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
    dev = _device(q)
    T, H = q.shape[0], q.shape[1]
    B = lens.shape[0]
    q_rs = _rows(q, "q", dev, T, H)
    ps, rs, hs, n_pages, page_size, HK = _pool(k_pages, v_pages, dev)
    if out is None:
        out = torch.empty((T, H, D), dtype=_BF16, device=q.device)
    o_rs = _rows(out, "out", dev, T, H)
    if T == 0:
        return out
    tab, tab_rs, tab_pages = _table(page_table, dev, B)
    most = tab_pages * page_size
    max_rows = T if max_rows is None or max_rows > T else max_rows
    max_keys = most if max_keys is None or max_keys > most else max_keys
    words, tree_ptr = 0, None
    if tree is not None:
        if (tree.dtype is not _I64T or tree.dim() != 2 or tree.shape[0] < T or not tree.is_contiguous()
                or tree.get_device() != dev):
            _refuse("tree", f"contiguous int64 [{T}, words]", tree)
        words, tree_ptr = tree.shape[1], tree.data_ptr()
    if window > INT_MAX or sinks > INT_MAX:
        raise ValueError("attention: window and sinks are 32-bit numbers")
    need = _ws_bytes(B, T, max_rows, max_keys, H, HK, page_size, window, sinks)
    ws, nbytes = None, 0
    if workspace is not None:
        nbytes = workspace.numel() * workspace.element_size()
        if nbytes < need or workspace.get_device() != dev or not workspace.is_contiguous():
            raise ValueError(f"workspace: {need} contiguous bytes on the current device needed")
        ws = workspace.data_ptr()
    elif need:
        workspace, nbytes = torch.empty(need, dtype=torch.uint8, device=q.device), need
        ws = workspace.data_ptr()
    _check("lr_cache_attention_bf16", lib().lr_cache_attention_bf16(
        q.data_ptr(), q_rs, out.data_ptr(), o_rs, k_pages.data_ptr(), v_pages.data_ptr(), ps, rs, hs, n_pages, page_size, tab,
        tab_rs, tab_pages, _ints(starts, "starts", dev, B + 1), _ints(lens, "lens", dev, B), B, T, max_rows, max_keys, H, HK,
        tree_ptr, words, window, sinks, scale, ws, nbytes, _raw_stream(dev)))
    return out


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """lr_cache_copy_pages: page src[i] to page dst[i] (int32 [n] on the device) in every layer of [layers, n_pages, page_size,
    heads, 128] (or one layer's pool). No target may occur twice or be a source."""
    dev = _device(k_pages)
    n = src.shape[0]
    pool = _pool(k_pages, v_pages, dev, True)
    if dst.shape[0] != n:
        raise ValueError("copy_pages: src and dst of different lengths")
    if n:
        _check("lr_cache_copy_pages", lib().lr_cache_copy_pages(
            k_pages.data_ptr(), v_pages.data_ptr(), *pool, _ints(src, "src", dev, n), _ints(dst, "dst", dev, n), n,
            _raw_stream(dev)))


def move_rows(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
              src: torch.Tensor, dst: torch.Tensor, *, max_rows: int | None = None) -> None:
    """lr_cache_move_rows: for the moves starts[b] .. starts[b + 1] of sequence b, its position src[i] to its position dst[i],
    in every layer; a sequence's rows are all read before any is written. max_rows: the most moves of a sequence (at most 256;
    default all of them)."""
    dev = _device(k_pages)
    n, B = src.shape[0], starts.shape[0] - 1
    pool = _pool(k_pages, v_pages, dev, True)
    if dst.shape[0] != n:
        raise ValueError("move_rows: src and dst of different lengths")
    if n:
        _check("lr_cache_move_rows", lib().lr_cache_move_rows(
            k_pages.data_ptr(), v_pages.data_ptr(), *pool, *_table(page_table, dev, B), _ints(starts, "starts", dev, B + 1),
            _ints(src, "src", dev, n), _ints(dst, "dst", dev, n), B, n, n if max_rows is None or max_rows > n else max_rows,
            _raw_stream(dev)))


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
        if any(self.holders[p] < n for p, n in collections.Counter(pages).items()):
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
