"""How attention cuts its work over blocks, on the CPU: every tile of every item is in exactly one segment, the blocks of a cut item
are those that its bookkeeping says, and no two partial results share a place."""
import ctypes as C
import os
import subprocess
import tempfile
from collections import defaultdict

import numpy as np
import pytest

from conftest import ROOT

LEAST = 16


@pytest.fixture(scope="module")
def shim():
    out = os.path.join(tempfile.mkdtemp(prefix="attention_plan"), "shim.so")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", out, os.path.join(ROOT, "tests", "attention_plan_shim.cpp")])
    lib = C.CDLL(out)
    lib.shim_attention_plan.restype = C.c_uint64
    lib.shim_attention_plan.argtypes = [C.c_void_p, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint32, C.c_void_p, C.c_uint64]
    return lib


def _plan(lib, lengths, items, blocks, shift=0):
    lengths = np.asarray(lengths, dtype=np.int64)
    out = np.zeros((300000, 7), dtype=np.uint64)
    n = lib.shim_attention_plan(lengths.ctypes.data, len(lengths), items, blocks, LEAST >> shift, shift, out.ctypes.data, len(out))
    assert n < len(out)
    return out[:n].astype(np.int64)


CASES = [([1], 1), ([37], 4), ([0, 0, 5, 0], 4), ([262144], 4), ([8200], 4), ([16] * 40, 2), ([17, 1, 0, 5000, 31], 3), ([0] * 600 + [40] + [0] * 500 + [1000], 8),
         (list(range(500, 8000, 233)), 4), ([100] * 256, 8), ([3100 + 16 * i for i in range(128)], 8), ([1], 148), ([1], 149), ([1] * 74, 1), ([5000] * 75, 1), ([2147483647], 2), ([2147483647], 31), ([262144] * 511, 512)]


@pytest.mark.parametrize("blocks", [1, 2, 7, 132, 148, 160])
@pytest.mark.parametrize("lengths,items", CASES)
@pytest.mark.parametrize("shift", [0, 2])
def test_every_tile_once_and_partial_results_apart(shim, lengths, items, blocks, shift):
    plan = _plan(shim, lengths, items, blocks, shift)
    by_item, places, owned = defaultdict(list), set(), defaultdict(set)
    for block, s, item, begin, end, owner, count in plan.tolist():
        assert end > begin
        by_item[(s, item)].append((begin, end, block, owner, count))
    assert set(by_item) == {(s, i) for s, n in enumerate(lengths) if n > 0 for i in range(items)}
    for (s, item), parts in by_item.items():
        assert [p[2] for p in parts] == sorted(p[2] for p in parts)
        assert parts[0][0] == 0 and parts[-1][1] == -(-lengths[s] // (16 << shift))
        assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
        if len(parts) == 1:
            continue
        assert {p[4] for p in parts} == {len(parts)} and {p[3] for p in parts} == {parts[0][2]}
        assert [p[2] for p in parts] == list(range(parts[0][3], parts[0][3] + len(parts)))
        owned[parts[0][3]].add((s, item))
        for p in parts:
            place = (p[2], p[2] == p[3])
            assert place not in places
            places.add(place)
    assert all(len(v) == 1 for v in owned.values())  # a block's counter serves one item


def test_few_items_are_cut_evenly(shim):
    plan = _plan(shim, [262144], 4, 148)
    sizes = plan[:, 4] - plan[:, 3]
    assert len(plan) == 144 and sizes.max() - sizes.min() <= 1
    plan = _plan(shim, [37], 4, 148)  # short items are not cut
    assert len(plan) == 4 and set(plan[:, 6]) == {1}
    plan = _plan(shim, [5000] * 75, 1, 148)
    sizes = np.bincount(plan[:, 0], weights=plan[:, 4] - plan[:, 3])
    assert sizes.max() - np.sort(sizes)[1] <= 1  # equal runs but for the last one


def test_short_items_stay_whole(shim):
    plan = _plan(shim, [60] * 28, 4, 148)  # 112 items of four tiles: a block each
    assert len(plan) == 112 and len(set(plan[:, 0])) == 112 and set(plan[:, 6]) == {1}
    plan = _plan(shim, [100] * 300, 8, 148)
    assert set(plan[:, 6]) == {1}
    sizes = np.bincount(plan[:, 0], weights=plan[:, 4] - plan[:, 3], minlength=148)
    run = -(-300 * 8 * 7 // 148)  # (the last block has what is left)
    assert sizes.max() <= run + 7 and np.sort(sizes)[1] >= run - 7 and sizes.sum() == 300 * 8 * 7


def test_division_by_page_size(shim):
    rng = np.random.default_rng(3)
    for per in [1, 2, 3, 4, 5, 6, 7, 12, 16, 31, 33, 1000, 4095, 65535, 65536]:
        tiles = [0, 1, per - 1, per, per + 1, 2 ** 27 - 1, 2 ** 27 - per] + rng.integers(0, 2 ** 27, 200).tolist()
        tiles += [per * k + d for k in rng.integers(1, 2 ** 27 // per, 50).tolist() for d in (-1, 0)]
        for t in tiles:
            for shift in (0, 2):
                assert shim.shim_attention_page_of((16 << shift) * per, shift, int(t)) == t // per
