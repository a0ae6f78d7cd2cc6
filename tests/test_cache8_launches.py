"""Which kernels attention_f8's sizes lead to, on the CPU: what the tests on the GPU run over the same sizes."""
from __future__ import annotations

import pytest

from tests.launch_util import LAUNCHES8, attention_f8


@pytest.mark.parametrize("sizes,want", LAUNCHES8, ids=str)
def test_launches(sizes, want):
    got = attention_f8(*sizes)
    assert {x: got[x] for x in want} == want
