"""Attention over packed prompts on the CPU: bad arguments are refused before any GPU call. No compute calls."""
from __future__ import annotations

import pytest
import torch

from localrouter_amd import _lib, ops

BAD = 1   # hipErrorInvalidValue
Q, K, V, O, S = (x << 32 for x in (1, 2, 3, 4, 8))   # fake, well-aligned device addresses, far apart from each other


def _packed(**kw):
    a = dict(q=Q, k=K, v=V, out=O, starts=S, B=3, T=300, H=8, HK=2, window=0, sinks=0, scale=0.088, qrs=1024, krs=256, vrs=256, ors=1024,
             stream=None)
    a.update(kw)
    return _lib.load().lr_attention_packed_bf16(*a.values())


@pytest.mark.parametrize("kw", [
    dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(starts=0), dict(starts=S + 2), dict(B=0), dict(B=65536), dict(T=0), dict(T=(1 << 28) + 1),
    dict(H=9), dict(HK=0), dict(H=0), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("inf")), dict(q=Q + 8),
    dict(qrs=1000), dict(krs=128), dict(vrs=252), dict(ors=1020), dict(krs=1 << 23), dict(vrs=1 << 23), dict(out=Q), dict(out=K + 4096),
    dict(out=V + 256),
], ids=str)
def test_packed_refuses(kw):
    assert _packed(**kw) == BAD


def test_tensors_on_the_host_are_refused():
    x, i = torch.zeros(3, 2, 128, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention_packed(x, x, x, i)
