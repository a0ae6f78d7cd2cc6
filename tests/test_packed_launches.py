"""Which kernel attention_packed's sizes lead to, on the CPU: blocks of 16 or 32 rows, or the stream of blocks of 128 or 256. Times of both
sides stand beside the rule (cache_abi.hip, packed_cut)."""
from __future__ import annotations

import pytest

from tests.launch_util import WINDOWED, WINDOWS, attention_packed

PROMPTS = [   # prompts, tokens, heads, kv heads: rows a block
    ((1, 1000, 1, 1), 16), ((1, 300, 32, 8), 32), ((1, 500, 32, 8), 32), ((2, 891, 32, 8), 128), ((1, 7000, 4, 1), 32), ((1, 4000, 8, 2), 32),
    ((2, 8000, 4, 1), 32), ((1, 8000, 1, 1), 32), ((1, 16000, 4, 1), 128), ((4, 12000, 4, 1), 128), ((20, 6000, 32, 8), 256),
    ((1, 16000, 32, 8), 256), ((3, 15000, 16, 16), 128), ((18, 611, 16, 8), 128),
]


def rows(*sizes, **kw):
    got = attention_packed(*sizes, **kw)
    return got["br"] or 32 * got["waves"]


@pytest.mark.parametrize("sizes,want", PROMPTS, ids=str)
def test_whole_prompts(sizes, want):
    assert rows(*sizes) == want
    # a window that hides nothing changes nothing
    assert rows(*sizes, window=sizes[1], sinks=4) == want and rows(*sizes, window=1 << 30, sinks=(1 << 31) - 1) == want


@pytest.mark.parametrize("sizes,window,sinks,want", [
    # few long prompts: the stream's blocks read a window, not all there is before them
    ((1, 7000, 4, 1), 64, 0, 128), ((1, 7000, 4, 1), 256, 4, 128), ((1, 7000, 4, 1), 1024, 4, 128), ((1, 4000, 8, 2), 64, 0, 128),
    ((1, 4000, 8, 2), 1024, 4, 128), ((2, 8000, 4, 1), 64, 0, 128), ((2, 8000, 4, 1), 1024, 4, 128), ((1, 500, 32, 8), 64, 0, 128),
    # one head: a round of blocks of 32 is all
    ((1, 8000, 1, 1), 64, 0, 32), ((1, 8000, 1, 1), 256, 4, 32), ((1, 8000, 1, 1), 1024, 4, 32), ((1, 1000, 1, 1), 64, 0, 16),
    # many blocks: as without a window
    ((20, 6000, 32, 8), 64, 0, 256), ((3, 15000, 16, 16), 256, 4, 128),
], ids=str)
def test_windows(sizes, window, sinks, want):
    assert rows(*sizes, window=window, sinks=sinks) == want


@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_what_the_gpu_runs(window, sinks):
    for lens, H, HK, want in WINDOWED:
        assert rows(len(lens), sum(lens), H, HK, window=window, sinks=sinks) == want
