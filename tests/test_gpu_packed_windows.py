"""attention_packed under windows and first tokens in each of its kernels, at sizes where the window is a small part of a prompt, against 64
bits."""
from __future__ import annotations

import pytest
import torch

from localrouter_amd import ops
from tests.cache_util import gen, rnd
from tests.launch_util import WINDOWED, WINDOWS
from tests.test_gpu_packed import check, ints, sums

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,H,HK,rows", WINDOWED, ids=lambda x: str(x) if isinstance(x, int) else f"{len(x)}x{x[0]}")
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_windows(lens, H, HK, rows, window, sinks):
    """(Blocks of `rows` rows: tests/test_packed_launches.py.)"""
    g, T = gen(41), sum(lens)
    q, k, v = rnd(g, T, H, 128), rnd(g, T, HK, 128), rnd(g, T, HK, 128)
    out = ops.attention_packed(q, k, v, ints(sums(lens)), window=window, sinks=sinks)
    check(q, k, v, out, lens, window, sinks, most=3)
    assert torch.equal(out, ops.attention_packed(q, k, v, ints(sums(lens)), window=window, sinks=sinks))
