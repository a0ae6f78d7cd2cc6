"""ctypes mirror of include/lr_cache.h and lr_cache8.h for torch tensors: a key / value cache in pages.

    append(q, k, v, k_pages, v_pages, page_table, starts, lens, ...)   norms, rotation and the write of new tokens, one pass
    attention(q, k_pages, v_pages, page_table, starts, lens, ...)      decode steps, chunks, drafted trees, windows
    copy_pages(k_pages, v_pages, src, dst)                             pages copied inside the pool, in every layer
    move_rows(k_pages, v_pages, page_table, starts, src, dst, ...)     rows moved inside their sequences, in every layer
    append_f8, attention_f8, copy_pages_f8                             the same over pages in 8 bits
    PagePool(n_pages)                                                  which pages are free, and who shares one (host only)

k_pages / v_pages: bf16 [n_pages, page_size, heads, 128] (copy_pages and move_rows also [layers, ...]), the same strides in
both; a pool laid out head by head is the permuted view of [n_pages, heads, page_size, 128]. page_table: int32 [B, pages a
sequence]; starts: int32 [B + 1], the call's tokens of sequence b being rows starts[b] .. starts[b + 1]; lens: int32 [B], the
sequences' lengths with those tokens. All on the current device.

Pages in 8 bits: float8_e4m3fn of the same shape (page_size 16 or more), and k_scales / v_scales: float8_e8m0fnu
[n_pages, page_size / 16, heads], its last two dimensions contiguous: the power of two of 16 rows of a page and head. What a pool holds
is pages.float() * scales.float().repeat_interleave(16, 1)[..., None].

Every call checks its tensors on the host (native/host_calls.cpp), then goes through the C ABI on torch's current HIP stream. There
is no fallback: without the built library every call raises.
"""
from __future__ import annotations

import collections
import ctypes
from pathlib import Path

import torch

from . import _lib
from .ops import PAIR_INTERLEAVED, SCALE_128, TABLE_COSSIN_F32, TABLE_NONE

HEADER = Path(__file__).resolve().parent.parent / "include" / "lr_cache.h"
HEADER_F8 = HEADER.with_name("lr_cache8.h")

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

SIGNATURES_F8 = {
    "lr_cache_append_f8": (_I, [_P, _P, _P, _I64, _I64, _I64, _P, _I64, _P, _P, _I64, _I64, _I64, _I, _I, _P, _P, _I64, _P, _I64, _I,
                                _P, _P, _P, _I, _I, _I, _I, _P, _P, _I, _P, _P, _I64, _I, _I, _I, _F, _P]),
    "lr_cache_attention_f8_ws_bytes": (_SZ, [_I] * 9),
    "lr_cache_attention_f8": (_I, [_P, _I64, _P, _I64, _P, _P, _I64, _I64, _I64, _I, _I, _P, _P, _I64, _P, _I64, _I, _P, _P, _I, _I,
                                   _I, _I, _I, _I, _P, _I, _I, _I, _F, _P, _SZ, _P]),
    "lr_cache_copy_pages_f8": (_I, [_P, _P, _I, _I64, _I64, _I64, _I64, _I, _I, _I, _P, _P, _I64, _I64, _P, _P, _I, _P]),
}

_bound = None
_calls = None
_current, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def lib() -> ctypes.CDLL:
    global _bound
    if _bound is None:
        L = _lib.load()
        for name, (res, args) in (SIGNATURES | SIGNATURES_F8).items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _bound = L
    return _bound


def _host():
    """The host side of the calls (native/host_calls.cpp), given the library's addresses at the first call."""
    global _calls
    if _calls is None:
        try:
            from . import _host_calls
        except ImportError as e:
            raise RuntimeError("localrouter_amd._host_calls is missing: build it with `python -m localrouter_amd.build` where torch and "
                               "Python's headers are installed (there is no fallback path)") from e
        L = lib()
        names = [*SIGNATURES, *SIGNATURES_F8, "lr_attention_window_bf16", "lr_attention_window_ws_bytes", "lr_attention_packed_bf16"]
        _host_calls.bind(_lib.LrError, {n: ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in names})
        _calls = _host_calls
    return _calls


def _device(t: torch.Tensor) -> int:
    """The current device; a host tensor is refused (there may be no device to ask)."""
    if not t.is_cuda:
        raise ValueError(f"expected tensors on the GPU, got one on {t.device}")
    return _current()


def append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
           page_table: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, q_out: torch.Tensor | None = None, *,
           q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, table_kind: int = TABLE_COSSIN_F32,
           table: tuple | None = None, positions: torch.Tensor | None = None, pairing: int = PAIR_INTERLEAVED, rot: int = 128,
           eps: float = 1e-6) -> torch.Tensor | None:
    """lr_cache_append_bf16: new tokens q [T, H, 128], k / v [T, HK, 128] (views of a packed projection allowed): queries
    normalised and rotated into q_out (allocated when None; q itself is allowed), keys the same way into their pages, values
    as they are. table = (table_a, table_b), one row a position, of rot / 2 columns at least (cos and sin) or 2 rot (2x2 kinds);
    positions int32 [T]: each token's table row (default its position in its sequence). q None: keys and values only. Returns q_out."""
    dev = _device(k_pages)
    if table is None:
        if table_kind != TABLE_NONE:
            raise ValueError("append: table required")
        table = (None, None)
    return (_calls or _host()).append(dev, _raw_stream(dev), q, k, v, k_pages, v_pages, page_table, starts, lens, q_out, q_norm,
                                      k_norm, table_kind, table[0], table[1], positions, pairing, rot, eps)


def attention_ws_bytes(B: int, T: int, max_rows: int, max_keys: int, heads: int, kv_heads: int, page_size: int, *,
                       window: int = 0, sinks: int = 0) -> int:
    """lr_cache_attention_ws_bytes: the workspace that a call with these numbers needs (0: none); smaller ones may need more."""
    return int(lib().lr_cache_attention_ws_bytes(*_lib.int32(B=B, T=T, max_rows=max_rows, max_keys=max_keys, heads=heads,
                                                             kv_heads=kv_heads, page_size=page_size, window=window, sinks=sinks)))


def attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
              lens: torch.Tensor, out: torch.Tensor | None = None, *, max_rows: int | None = None,
              max_keys: int | None = None, tree: torch.Tensor | None = None, window: int = 0, sinks: int = 0,
              scale: float = SCALE_128, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """lr_cache_attention_bf16: the batch's tokens q [T, H, 128] over their sequences' pages (append first). The token at
    position p sees positions j <= p; with tree (int64 [T, words], bit x of a token's words: it sees the sequence's x-th token
    of the call) drafted tokens see everything before the call's tokens and what their bits say. window n >= 1: earlier
    positions (under a tree: those before the call's tokens) only where p - j < n or j < sinks. max_rows: the most tokens of a
    sequence; max_keys: the longest sequence. Both choose the kernel and size the launch, which has workgroups for max_rows tokens of
    every sequence: give them. Their defaults, all T tokens and what the table holds, are for single sequences; of a batch most
    workgroups are without rows then, and where a grid does not hold them the call is refused. A workspace of attention_ws_bytes
    for the same numbers is allocated when none is given."""
    dev = _device(q)
    return (_calls or _host()).attention(dev, _raw_stream(dev), q, k_pages, v_pages, page_table, starts, lens, out, max_rows, max_keys,
                                         tree, window, sinks, scale, workspace)


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """lr_cache_copy_pages: page src[i] to page dst[i] (int32 [n] on the device) in every layer of [layers, n_pages, page_size,
    heads, 128] (or one layer's pool). No target may occur twice or be a source."""
    dev = _device(k_pages)
    (_calls or _host()).copy_pages(dev, _raw_stream(dev), k_pages, v_pages, src, dst)


def move_rows(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
              src: torch.Tensor, dst: torch.Tensor, *, max_rows: int | None = None) -> None:
    """lr_cache_move_rows: for the moves starts[b] .. starts[b + 1] of sequence b, its position src[i] to its position dst[i],
    in every layer; a sequence's rows are all read before any is written. No position may be a target
    twice. max_rows: the most moves of a sequence (at most 256; default all of them)."""
    dev = _device(k_pages)
    (_calls or _host()).move_rows(dev, _raw_stream(dev), k_pages, v_pages, page_table, starts, src, dst, max_rows)


def append_f8(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              k_scales: torch.Tensor, v_scales: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor,
              q_out: torch.Tensor | None = None, *, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
              table_kind: int = TABLE_COSSIN_F32, table: tuple | None = None, positions: torch.Tensor | None = None,
              pairing: int = PAIR_INTERLEAVED, rot: int = 128, eps: float = 1e-6) -> torch.Tensor | None:
    """lr_cache_append_f8: append() into pages in 8 bits. Keys and values are rounded once, from fp32, to the scale of their 16 rows, the
    least power of two that holds the call's rows among them; where earlier positions of the sequence lie among them it is no less
    than before, and if it rises their rows are rounded again. An infinity or NaN is held as NaN and has no part in the scale."""
    dev = _device(k_pages)
    if table is None:
        if table_kind != TABLE_NONE:
            raise ValueError("append_f8: table required")
        table = (None, None)
    return (_calls or _host()).append_f8(dev, _raw_stream(dev), q, k, v, k_pages, v_pages, page_table, starts, lens, q_out, q_norm,
                                         k_norm, table_kind, table[0], table[1], positions, pairing, rot, eps, k_scales, v_scales)


def attention_f8_ws_bytes(B: int, T: int, max_rows: int, max_keys: int, heads: int, kv_heads: int, page_size: int, *,
                          window: int = 0, sinks: int = 0) -> int:
    """lr_cache_attention_f8_ws_bytes: the workspace that attention_f8 with these numbers needs (0: none); smaller ones may need more."""
    return int(lib().lr_cache_attention_f8_ws_bytes(*_lib.int32(B=B, T=T, max_rows=max_rows, max_keys=max_keys, heads=heads,
                                                                kv_heads=kv_heads, page_size=page_size, window=window, sinks=sinks)))


def attention_f8(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                 page_table: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, out: torch.Tensor | None = None, *,
                 max_rows: int | None = None, max_keys: int | None = None, tree: torch.Tensor | None = None, window: int = 0,
                 sinks: int = 0, scale: float = SCALE_128, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """lr_cache_attention_f8: attention() over pages in 8 bits; queries, probabilities and the output are bf16."""
    dev = _device(q)
    return (_calls or _host()).attention_f8(dev, _raw_stream(dev), q, k_pages, v_pages, page_table, starts, lens, out, max_rows,
                                            max_keys, tree, window, sinks, scale, workspace, k_scales, v_scales)


def copy_pages_f8(k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor, src: torch.Tensor,
                  dst: torch.Tensor) -> None:
    """lr_cache_copy_pages_f8: copy_pages() of pages in 8 bits and their scales ([layers, ...] in both or in neither)."""
    dev = _device(k_pages)
    (_calls or _host()).copy_pages_f8(dev, _raw_stream(dev), k_pages, v_pages, k_scales, v_scales, src, dst)


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
