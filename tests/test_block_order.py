"""The order in which an XCD's blocks of rows start (localrouter_amd/csrc/block_order.h), compiled for the host: against a model of the
places that they start on."""
from __future__ import annotations

import ctypes
import heapq
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "localrouter_amd" / "csrc"
CUS = 32


@pytest.fixture(scope="module")
def order(tmp_path_factory):
    d = tmp_path_factory.mktemp("order")
    (d / "o.cpp").write_text('#include "block_order.h"\nextern "C" int order(int i, int n, int c) { return lr::start_order(i, n, c); }\n')
    subprocess.run([shutil.which("g++") or "g++", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", str(d / "o.cpp"), "-o", str(d / "o.so")],
                   check=True)
    lib = ctypes.CDLL(str(d / "o.so"))
    return lambda n, per_cu: [lib.order(i, n, per_cu) for i in range(n)]


def end_of(order, cost, per_cu):
    """When the last block ends: workgroups start in order on the place that is free first; those of one CU take turns (two blocks of
    4 waves side by side take as long as one after the other)."""
    if per_cu == 2:
        assert len(order) <= 2 * CUS
        return max(sum(cost[b] for b in order[cu::CUS]) for cu in range(CUS))
    free = [0.0] * CUS
    for b in order:
        heapq.heapreplace(free, free[0] + cost[b])
    return max(free)


@pytest.mark.parametrize("per_cu", [1, 2])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 40, 63, 64, 65, 100, 128, 500])
def test_every_block_starts_once(order, n, per_cu):
    assert sorted(order(n, per_cu)) == list(range(n))


@pytest.mark.parametrize("n", [33, 34, 48, 63, 64])
@pytest.mark.parametrize("before", [0, 16, 64])
def test_blocks_of_causal_rows_end_no_later_than_in_the_other_order(order, n, before):
    """Blocks of causal rows, longest first, behind `before` tiles of keys: key tiles and four tiles of start and end each. One workgroup
    a CU: longest first throughout. Two: the second of a CU in the opposite order."""
    cost = [4 + before + (n - b) * 64 / n for b in range(n)]
    plain = list(range(n))
    other = plain[:32] + plain[32:][::-1]
    one, two = order(n, 1), order(n, 2)
    assert end_of(one, cost, 1) <= min(end_of(plain, cost, 1), end_of(other, cost, 1))
    assert end_of(two, cost, 2) <= min(end_of(plain, cost, 2), end_of(other, cost, 2))
    if n == 64:
        assert end_of(other, cost, 1) > 1.08 * end_of(one, cost, 1)
