"""What the workspaces of the attention over pages amount to (INTEGRATION's figures): host arithmetic, no GPU."""
from __future__ import annotations

import random

import pytest

from localrouter_amd import cache

ROW = 520   # bytes of a row of a part: 128 sums, its reference and its sum
MOST = 8 * 64 * 4 * 256 * ROW + 4096   # 8 XCDs x 64 pieces x 4 blocks of 256 rows


def need(f, B, rows, keys, H, HK, ps, **kw):
    return f(B, B * rows, rows, keys, H, HK, ps, **kw)


@pytest.mark.parametrize("ps", [16, 32, 256])
@pytest.mark.parametrize("f,entries", [(cache.attention_ws_bytes, 2048), (cache.attention_f8_ws_bytes, 1024)], ids=["bf16", "f8"])
def test_ranges_whose_entries_a_workgroup_holds(f, entries, ps):
    """Calls are cut only where that fills the GPU, into at most as many parts as it has places."""
    rng = random.Random(ps)
    limit, top = entries * min(ps, 32), 0
    for _ in range(20000):
        B, HK, G = int(2 ** rng.uniform(0, 10)), rng.choice([1, 2, 3, 8, 16, 32]), rng.choice([1, 2, 4, 7, 16])
        rows, keys = int(2 ** rng.uniform(0, 14)), min(limit, int(2 ** rng.uniform(4, 17)))
        if B * rows * G * HK > 1 << 22:
            continue
        window = rng.choice([0, 0, int(2 ** rng.uniform(0, 14))])
        top = max(top, need(f, B, rows, keys, G * HK, HK, ps, window=window, sinks=rng.choice([0, 4])))
    assert 100e6 < top <= MOST


@pytest.mark.parametrize("sizes,bf16,f8", [
    # sequences, tokens, positions, heads, kv heads, page: rows x parts
    ((8, 2048, 131072, 32, 8, 16), 8 * 2048 * 32 * 4, 8 * 2048 * 32 * 3),      # (bf16 in parts of 32,768 positions, f8 of 61,440)
    ((64, 512, 131072, 32, 8, 16), 64 * 512 * 32 * 4, 64 * 512 * 32 * 3),
    ((16, 2048, 131072, 64, 8, 16), 16 * 2048 * 64 * 4, 16 * 2048 * 64 * 3),
    ((8, 2048, 131072, 32, 8, 64), 8 * 2048 * 32 * 2, 0),                      # (of 65,536; of 245,760)
    ((16, 2048, 61441, 64, 8, 16), 16 * 2048 * 64 * 2, 16 * 2048 * 64 * 2),
    ((16, 2048, 61440, 64, 8, 16), 16 * 2048 * 64 * 2, 0),
    ((256, 1, 131072, 32, 8, 16), 256 * 8 * 16 * 4, 256 * 8 * 16 * 8),         # (of 32,768, of 16,384; 4 rows in blocks of 16)
], ids=str)
def test_longer_ranges_take_a_part_for_as_many_entries(sizes, bf16, f8):
    for f, rows in ((cache.attention_ws_bytes, bf16), (cache.attention_f8_ws_bytes, f8)):
        got = need(f, *sizes)
        assert rows * ROW <= got <= rows * ROW + rows // 16 * 8 + 1024   # (and flags, one a block and part)
