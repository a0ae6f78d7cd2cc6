"""The host side of the paged cache and of the packed attention (localrouter_amd/csrc/cache_abi.hip) built by itself for the CPU, with
launches that only write down what they were given: which kernel a call's sizes and layouts lead to, and which calls are refused. No
GPU call is made, whatever the addresses are."""
from __future__ import annotations

import ctypes
import subprocess
import tempfile
from pathlib import Path

from localrouter_amd import _lib as bindings
from localrouter_amd import build, cache

CSRC = Path(__file__).resolve().parent.parent / "localrouter_amd" / "csrc"
FIELDS = ("kernel", "br", "waves", "kh", "hw", "nsplit", "per", "places", "teams", "merge_here", "nblk")
KERNELS = {1: "step", 2: "wide", 3: "step packed", 4: "wide packed", 5: "step8", 6: "wide8", 7: "append", 8: "append8", 9: "copy",
           10: "scales"}

SOURCE = """
#include "cache_abi.hip"
static int64_t last[11];
static int launches;
static hipError_t note(int kernel, const lr::RangeAttnArgs& a, int br, int waves, int kh, int hw) {
    const int64_t x[11] = {kernel, br, waves, kh, hw, a.nsplit, a.per, a.places, a.teams, a.merge_here, a.nblk};
    std::copy(x, x + 11, last);
    ++launches;
    return hipSuccess;
}
static hipError_t note(int kernel) { return note(kernel, lr::RangeAttnArgs{}, 0, 0, 0, 0); }
namespace lr {
hipError_t launch_range_attn(const RangeAttnArgs& a, bool, int br, hipStream_t) { return note(1, a, br, 0, 0, 0); }
hipError_t launch_range_wide(const RangeAttnArgs& a, bool, int waves, hipStream_t) { return note(2, a, 0, waves, 0, 0); }
hipError_t launch_packed_attn(const RangeAttnArgs& a, int br, hipStream_t) { return note(3, a, br, 0, 0, 0); }
hipError_t launch_packed_wide(const RangeAttnArgs& a, int waves, hipStream_t) { return note(4, a, 0, waves, 0, 0); }
hipError_t launch_range8(const RangeAttnArgs& a, int br, int kh, int hw, hipStream_t) { return note(5, a, br, 0, kh, hw); }
hipError_t launch_range_wide8(const RangeAttnArgs& a, int waves, hipStream_t) { return note(6, a, 0, waves, 0, 0); }
hipError_t launch_cache_append(const CacheAppendArgs&, hipStream_t) { return note(7); }
hipError_t launch_cache_append8(const CacheAppend8Args&, hipStream_t) { return note(8); }
hipError_t launch_cache_copy(const CacheCopyArgs&, hipStream_t) { return note(9); }
hipError_t launch_cache_copy_scales(const CacheCopyScalesArgs&, hipStream_t) { return note(10); }
hipError_t launch_cache_move(const CacheMoveArgs&, hipStream_t) { return hipSuccess; }
}
extern "C" int launched(int64_t* to) {
    std::copy(last, last + 11, to);
    const int n = launches;
    launches = 0;
    return n;
}
"""

_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        with tempfile.TemporaryDirectory() as d:
            src, out = Path(d) / "l.hip", Path(d) / "l.so"
            src.write_text(SOURCE)
            subprocess.run([build.hipcc(), "--offload-host-only", "-x", "hip", "-O1", "-std=c++17", "-shared", "-fPIC", "-w", f"-I{CSRC}",
                            str(src), "-o", str(out)], check=True)
            L = ctypes.CDLL(str(out))
        for name, (res, args) in (cache.SIGNATURES | cache.SIGNATURES_F8).items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        L.lr_attention_packed_bf16.restype, L.lr_attention_packed_bf16.argtypes = bindings.SIGNATURES["lr_attention_packed_bf16"]
        _lib = L
    return _lib


def launch_of(name: str, *args) -> dict | None:
    """The last launch of the call (its sizes and choices by name), None where it is refused before any."""
    L = lib()
    x = (ctypes.c_int64 * len(FIELDS))()
    L.launched(x)
    rc = getattr(L, name)(*args)
    n = L.launched(x)
    assert (rc == 0) == (n > 0), (rc, n)
    if not n:
        return None
    return dict(zip(FIELDS, x), kernel=KERNELS[x[0]])


# attention_f8's sizes (sequences, max_rows, max_keys, heads, kv heads, page size) and the launches that they lead to: kernels whose batch
# is large, and parts that there are only because a workgroup holds so many entries of the page table (step8 1,024, wide8 3,840)
LAUNCHES8 = [
    ((100, 1, 400, 32, 8, 16), dict(kernel="step8", br=16, kh=2, hw=2, nsplit=1)),
    ((64, 1, 300, 64, 16, 32), dict(kernel="step8", br=16, kh=2, hw=2, nsplit=1)),
    ((100, 4, 400, 32, 8, 16), dict(kernel="step8", br=16, kh=2, hw=2, nsplit=1)),
    ((100, 1, 20000, 32, 8, 16), dict(kernel="step8", br=16, kh=2, hw=2, nsplit=2, per=512, merge_here=1)),
    ((100, 4, 16400, 32, 8, 16), dict(kernel="step8", br=16, kh=2, hw=2, nsplit=2, per=512, merge_here=1)),
    ((120, 1, 20000, 14, 7, 16), dict(kernel="step8", br=16, kh=4, hw=1, nsplit=2, per=512, merge_here=1)),
    ((20, 16, 20000, 32, 8, 16), dict(kernel="step8", br=32, kh=4, hw=1, nsplit=2, per=512, merge_here=0, nblk=2)),
    ((70, 6, 20000, 32, 8, 16), dict(kernel="step8", br=32, kh=4, hw=1, nsplit=2, per=512, merge_here=0, nblk=1)),
    ((1, 1200, 66000, 64, 1, 16), dict(kernel="wide8", waves=8, nsplit=2, per=960, places=0, teams=0)),
    ((24, 12, 66000, 256, 8, 16), dict(kernel="wide8", waves=4, nsplit=2, per=960, places=0, teams=0)),
]


def attention_f8(B, rows, keys, H, HK, ps, window=0, sinks=0) -> dict | None:
    """The launch of cache.attention_f8 for a batch of B x rows tokens."""
    q, out, kp, vp, ks, vs, table, starts, lens, ws = (x << 44 for x in range(1, 11))
    pages = -(-keys // ps)
    return launch_of("lr_cache_attention_f8", q, 128 * H, out, 128 * H, kp, vp, 128 * HK * ps, 128 * HK, 128, 1 << 16, ps, ks, vs,
                     ps // 16 * HK, table, pages, pages, starts, lens, B, B * rows, rows, keys, H, HK, None, 0, window, sinks, 0.088, ws,
                     1 << 43, None)


# attention_packed under windows: prompts, heads, kv heads, the rows of the blocks that every window of WINDOWS leads to
WINDOWED = [([1000], 1, 1, 16), ([8000], 1, 1, 32), ([7000], 4, 1, 128), ([4100, 3, 0, 3900], 4, 1, 128), ([1500, 1700] * 4, 32, 8, 256)]
WINDOWS = [(1, 0), (64, 0), (65, 3), (256, 4), (1000, 70)]


def attention_packed(B, T, H, HK, window=0, sinks=0) -> dict | None:
    """The launch of ops.attention_packed for T tokens of B prompts."""
    q, k, v, out, starts = (x << 44 for x in range(1, 6))
    return launch_of("lr_attention_packed_bf16", q, k, v, out, starts, B, T, H, HK, window, sinks, 0.088, 128 * H, 128 * HK, 128 * HK, 128 * H,
                     None)
