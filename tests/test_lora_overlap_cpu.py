"""Adapters whose output shares memory with what the call reads are refused before anything is launched; rows that
only lie between each other's are not. (Addresses that nothing reads: without a GPU a call that passes the checks ends
in a device error.)"""
import ctypes
import random

import pytest
import torch

from swarmllm_amd._lib import QMM_DEVICE_ERROR, QMM_UNSUPPORTED, X_BF16, X_F32, Adapter, lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="calls with addresses of nothing")
M = 1 << 24  # far apart


def call(rows, k, n, rank=8, slots=2, count=1, x=M, xs=None, ids=2 * M, ws=3 * M, **change):
    """A launch of `count` projections; y, out, a, b, scales (and the strides ys, os) by projection as lists or one."""
    c = (Adapter * 4)()
    for i in range(count):
        f = {"a": (4 + 8 * i) * M, "b": (5 + 8 * i) * M, "scales": (6 + 8 * i) * M, "y": (7 + 8 * i) * M,
             "out": (8 + 8 * i) * M, "ys": n, "os": n}
        for key, v in change.items():
            f[key] = v[i] if isinstance(v, list) else v
        c[i] = Adapter(f["a"], f["b"], f["scales"], f["y"], f["out"], n, f["ys"], f["os"], rank)
    need = ctypes.c_size_t()
    return lib().qmm_adapters_add(count, c, slots, X_BF16, x, X_F32, xs or k, ids, k, rows, ws, 1 << 40, ctypes.byref(need), 1, 0)


def test_everything_apart_or_in_place_is_taken():
    for rows in (1, 3, 2000):
        assert call(rows, 64, 50) == QMM_DEVICE_ERROR
        assert call(rows, 64, 50, y=9 * M, out=9 * M) == QMM_DEVICE_ERROR
        assert call(rows, 64, 50, count=3) == QMM_DEVICE_ERROR
        # three projections as columns of one wide array, in place, and x's columns beside them
        wide = [9 * M, 9 * M + 200, 9 * M + 400]
        assert call(rows, 64, 50, count=3, y=wide, out=wide, ys=214, os=214, x=9 * M + 600, xs=214) == QMM_DEVICE_ERROR


def test_shared_memory_is_refused():
    for rows in (1, 3, 2000):
        for off in (-4 * 49, -4, 4, 4 * 49):  # beside its own y without being it
            assert call(rows, 64, 50, y=9 * M, out=9 * M + off) == QMM_UNSUPPORTED, (rows, off)
        assert call(rows, 64, 50, out=M + 64) == QMM_UNSUPPORTED  # x
        assert call(rows, 64, 50, out=2 * M) == QMM_UNSUPPORTED  # ids
        assert call(rows, 64, 50, out=4 * M + 128) == QMM_UNSUPPORTED  # a
        assert call(rows, 64, 50, out=5 * M) == QMM_UNSUPPORTED  # b
        assert call(rows, 64, 50, out=6 * M + 4) == QMM_UNSUPPORTED  # scales
        # another projection's y and out
        assert call(rows, 64, 50, count=2, out=[9 * M, 9 * M + 4]) == QMM_UNSUPPORTED
        assert call(rows, 64, 50, count=2, y=[9 * M, 10 * M], out=[10 * M + 4, 11 * M]) == QMM_UNSUPPORTED
        wide = [9 * M, 9 * M + 196]
        assert call(rows, 64, 50, count=2, y=wide, out=wide, ys=214, os=214) == QMM_UNSUPPORTED
    assert call(2000, 64, 50, ws=M + 64) == QMM_UNSUPPORTED and call(2000, 64, 50, ws=2 * M) == QMM_UNSUPPORTED
    assert call(2000, 64, 50, out=3 * M) == QMM_UNSUPPORTED
    # strides past 2^62 values
    assert call(3, 64, 50, xs=2 ** 62, ys=2 ** 62, os=2 ** 62, out=7 * M) == QMM_DEVICE_ERROR


@pytest.mark.parametrize("seed", range(4))
def test_rows_between_rows(seed):
    rng = random.Random(seed)
    seen = set()
    for _ in range(1500):
        n, rows = rng.randint(1, 6), rng.randint(1, 6)
        ys, os_ = rng.randint(n, 20), rng.randint(n, 20)
        if rng.random() < 0.5:
            os_ = ys
        y, out = 64 * M + 4 * rng.randint(0, 90), 64 * M + 4 * rng.randint(0, 90)
        if y == out:
            continue
        cells = lambda at, s: {at // 4 + r * s + e for r in range(rows) for e in range(n)}
        shared = bool(cells(y, ys) & cells(out, os_))
        seen.add(shared)
        got = call(rows, 32, n, y=y, out=out, ys=ys, os=os_)
        assert got == (QMM_UNSUPPORTED if shared else QMM_DEVICE_ERROR), (n, rows, ys, os_, y, out)
    assert seen == {True, False}
