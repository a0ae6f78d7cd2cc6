"""Which layouts of the scales of 8-bit pages the calls take: all in which no two scales share a byte, and no others. On the CPU: the
host side alone, whose launches are written down (launch_util)."""
from __future__ import annotations

import itertools
import random

import pytest

from tests.launch_util import launch_of

KP, VP, SC, Q, OUT, WS, I1, I2, I3 = (x << 44 for x in (1, 2, 3, 4, 5, 6, 7, 8, 9))
HK, PAGE = 2, 32
BYTES = PAGE // 16 * HK   # of a page and layer


def copy(d, layers, sls, n_pages, sps):
    return launch_of("lr_cache_copy_pages_f8", KP, VP, layers, 1 << 24, PAGE * HK * 128, HK * 128, 128, n_pages, PAGE, HK, SC, SC + d, sls,
                     sps, I1, I2, 3, None)


def attend(d, n_pages, sps):
    return launch_of("lr_cache_attention_f8", Q, 1024, OUT, 1024, KP, VP, PAGE * HK * 128, HK * 128, 128, n_pages, PAGE, SC, SC + d, sps, I1,
                     4, 4, I2, I3, 1, 1, 1, 100, 8, HK, None, 0, 0, 0, 0.088, WS, 1 << 30, None)


def append(d, n_pages, sps):
    return launch_of("lr_cache_append_f8", None, Q, OUT, 256, 256, 256, None, 0, KP, VP, PAGE * HK * 128, HK * 128, 128, n_pages, PAGE, SC,
                     SC + d, sps, I1, 4, 4, I2, I3, None, 1, 20, 0, HK, None, None, 0, None, None, 0, 0, 0, 0, 1e-6, None)


# the outermost dimension first
@pytest.mark.parametrize("order", list(itertools.permutations(["layers", "kv", "pages"])), ids="-".join)
@pytest.mark.parametrize("layers,n_pages", [(3, 7), (1, 7), (3, 1), (2, 2)])
def test_scales_of_keys_values_layers_and_pages_side_by_side_in_any_order(order, layers, n_pages):
    count, st, at = dict(layers=layers, kv=2, pages=n_pages), {}, BYTES
    for name in reversed(order):
        st[name] = at
        at *= count[name]
    assert copy(st["kv"], layers, st["layers"], n_pages, st["pages"])["kernel"] == "scales"
    assert copy(-st["kv"], layers, st["layers"], n_pages, st["pages"])["kernel"] == "scales"
    # one layer's view of them
    assert attend(st["kv"], n_pages, st["pages"])["kernel"] == "step8"
    assert append(st["kv"], n_pages, st["pages"])["kernel"] == "append8"


def test_scales_are_refused_where_they_share_bytes_and_nowhere_else():
    """Random small layouts, nested in every order and not nested, against the bytes themselves."""
    rng = random.Random(5)
    some = [0, 0]
    for _ in range(3000):
        layers, n_pages = rng.choice([1, 2, 3, 5]), rng.choice([1, 2, 4, 9])
        dims = [["layers", layers], ["pages", n_pages], ["kv", 2]]
        rng.shuffle(dims)
        at, st = BYTES, {}
        for name, n in dims:
            st[name] = at
            at = at * n + rng.choice([0, 0, 0, 1, BYTES])
        if rng.random() < 0.5:
            st["kv"] = rng.choice([1, -1]) * rng.randrange(0, at + 2)
        if rng.random() < 0.3:
            st["layers"] = rng.randrange(1, at + 2)
        if rng.random() < 0.1:
            st["pages"] = rng.randrange(1, at + 2)
        held = [kv * st["kv"] + l * st["layers"] + p * st["pages"] + x for kv in (0, 1) for l in range(layers) for p in range(n_pages)
                for x in range(BYTES)]
        shared = len(set(held)) < len(held)
        some[shared] += 1
        if n_pages == 1 and st["pages"] < BYTES:
            continue   # (a stride of less than a page's scales is refused whether it is taken or not)
        assert (copy(st["kv"], layers, st["layers"], n_pages, st["pages"]) is None) == shared, (st, layers, n_pages)
        if layers == 1:
            assert (attend(st["kv"], n_pages, st["pages"]) is None) == shared, (st, n_pages)
            assert (append(st["kv"], n_pages, st["pages"]) is None) == shared, (st, n_pages)
    assert min(some) > 300
