"""The batch's C entries without a GPU: what they plan, and refusals before
anything touches the device. The plain implementations of the GPU tests against
cases counted by hand."""
import ctypes
import math

import pytest
import torch

import batch_reference as ref
from swarmllm_amd._lib import (QMM_NO_ROOM, QMM_OK, QMM_UNSUPPORTED, QMM_WORKSPACE_TOO_SMALL, X_BF16, X_F32, Adapter, Pages,
                               lib)

P = 4096  # a 16-byte aligned address that is never read


def pages_step(tokens=10, q=P, taken=P, slots=P, **change):
    p = Pages(P, P, P, P, 20, 20, 100, 8, 64)
    for k, v in change.items():
        setattr(p, k, v)
    return lib().qmm_pages_step(ctypes.byref(p), None, None, tokens, q, taken, slots, None, None, 0)


def test_pages_refusals():
    for bad in (dict(seqs=-1), dict(seqs=4097), dict(page=8), dict(page=48), dict(page=512), dict(page=0),
                dict(row_pages=-1), dict(table_stride=19), dict(pool=-1), dict(pool=2**31), dict(row_pages=2**24 + 1,
                table_stride=2**40), dict(seqs=4096, row_pages=2**19, table_stride=2**19),
                dict(seqs=1024, row_pages=2**10, table_stride=2**20 + 1), dict(tables=None),
                dict(lens=None), dict(free_pages=None), dict(free_count=None), dict(q=None), dict(taken=None),
                dict(slots=None), dict(tokens=-1), dict(tokens=2**29 + 1)):
        assert pages_step(**bad) == QMM_UNSUPPORTED, bad
    assert lib().qmm_pages_step(None, None, None, 0, P, P, P, None, None, 0) == QMM_UNSUPPORTED


def adapters_add(n=None, launch=0, count=1, slots=4, w=X_BF16, x=17 * P, x_type=X_F32, x_stride=4096, ids=P, k=4096, rows=5,
                 ws=None, ws_bytes=0, **change):
    c = (Adapter * 4)(*[Adapter(P, P, P, 9 * P + 4096 * i, P + 4096 * i, 1000, 1000, 1000, 16) for i in range(4)])
    for key, v in change.items():
        setattr(c[0], key, v)
    n = n if n is not None else ctypes.c_size_t(7)
    return lib().qmm_adapters_add(count, c, slots, w, x, x_type, x_stride, ids, k, rows, ws, ws_bytes, ctypes.byref(n),
                                  launch, 0), n.value


def test_adapters_plan_and_refusals():
    assert adapters_add() == (QMM_OK, 0)  # few rows of a short k: in one launch, nothing between
    st, need = adapters_add(rows=3000)
    assert st == QMM_OK and need >= 3000 * 16 * 4
    assert adapters_add(k=28672, x_stride=28672)[1] >= 5 * 16 * 4
    many = [adapters_add(rows=2000, slots=s)[1] for s in (1, 4, 100)]
    assert 2000 * 16 * 4 <= many[0] < many[1] < many[2]  # whole tiles, and one begun for each adapter
    assert adapters_add(rows=0) == (QMM_OK, 0) and adapters_add(rows=0, launch=1) == (QMM_OK, 0)
    assert adapters_add(rows=3000, launch=1, ws=P, ws_bytes=need - 1) == (QMM_WORKSPACE_TOO_SMALL, need)
    assert adapters_add(rows=3000, launch=1)[0] == QMM_WORKSPACE_TOO_SMALL
    assert adapters_add(launch=1, ws=P + 4, ws_bytes=2 * need)[0] == QMM_UNSUPPORTED
    for bad in (dict(count=0), dict(count=5), dict(slots=-1), dict(slots=4097), dict(w=3), dict(x_type=-1), dict(x_stride=4095), dict(k=0),
                dict(k=4080 + 8), dict(rows=-1), dict(rows=2**20 + 1), dict(n=ctypes.c_size_t(), rank=0), dict(rank=12),
                dict(rank=136), dict(y_stride=999), dict(out_stride=999), dict(y=P, out=P, out_stride=1004), dict(a=P + 8),
                dict(b=P + 4)):
        assert adapters_add(**bad)[0] == QMM_UNSUPPORTED, bad
    # two projections into one place, and more workgroups than a launch takes
    assert adapters_add(count=2)[0] == QMM_OK and adapters_add(count=2, out=2 * P)[0] == QMM_UNSUPPORTED
    assert adapters_add(count=2, out=10 * P)[0] == QMM_UNSUPPORTED and adapters_add(count=2, y=2 * P)[0] == QMM_UNSUPPORTED
    assert adapters_add(x=5 * P, out=5 * P)[0] == QMM_UNSUPPORTED
    wide = dict(n=2**30, y_stride=2**31, out_stride=2**31)
    c = (Adapter * 1)(Adapter(P, P, P, P, P, wide["n"], wide["y_stride"], wide["out_stride"], 16))
    assert lib().qmm_adapters_add(1, c, 4, X_BF16, 17 * P, X_F32, 4096, P, 4096, 1, None, 0, ctypes.byref(ctypes.c_size_t()), 0,
                                  0) == QMM_OK
    assert lib().qmm_adapters_add(1, c, 4, X_BF16, 17 * P, X_F32, 4096, P, 4096, 64, None, 0, ctypes.byref(ctypes.c_size_t()), 0,
                                  0) == QMM_UNSUPPORTED
    for null in (dict(x=None), dict(ids=None), dict(a=None), dict(b=None), dict(y=None), dict(out=None)):
        assert adapters_add(launch=1, ws=P, ws_bytes=2**20, **null)[0] == QMM_UNSUPPORTED, null
    st = lib().qmm_adapters_add(1, (Adapter * 1)(), 1, 0, P, 0, 4096, P, 4096, 1, None, 0, None, 0, 0)
    assert st == QMM_UNSUPPORTED


def sample(launch=0, logits=P, dtype=X_F32, stride=1000, u=P, ids=P, vocab=1000, rows=3, ws=None, ws_bytes=0):
    n = ctypes.c_size_t(7)
    return lib().qmm_sample(logits, dtype, stride, u, None, None, None, None, ids, None, vocab, rows, ws, ws_bytes,
                            ctypes.byref(n), launch, 0), n.value


def test_sample_plan_and_refusals():
    st, need = sample()
    assert st == QMM_OK and need > 0
    assert sample(rows=0) == (QMM_OK, 0) and sample(rows=0, launch=1) == (QMM_OK, 0)
    assert sample(launch=1, ws=P, ws_bytes=need - 1) == (QMM_WORKSPACE_TOO_SMALL, need)
    assert sample(launch=1, ws=P + 8, ws_bytes=2 * need)[0] == QMM_UNSUPPORTED
    for bad in (dict(dtype=3), dict(stride=999), dict(vocab=0), dict(vocab=2**19 + 1, stride=2**20), dict(rows=-1),
                dict(rows=65536)):
        assert sample(**bad)[0] == QMM_UNSUPPORTED, bad
    for null in (dict(logits=None), dict(u=None), dict(ids=None)):
        assert sample(launch=1, ws=P, ws_bytes=2 * need, **null)[0] == QMM_UNSUPPORTED, null
    assert lib().qmm_sample(P, 0, 10, P, None, None, None, None, P, None, 10, 1, None, 0, None, 0, 0) == QMM_UNSUPPORTED


def test_injected_failure_is_one_call_s():
    need = sample()[1]
    lib().qmm_fail_next_launch()
    assert sample(launch=1, ws=P, ws_bytes=need)[0] == QMM_NO_ROOM
    assert sample(launch=1, ws=P, ws_bytes=0)[0] == QMM_WORKSPACE_TOO_SMALL
    lib().qmm_fail_next_launch()
    assert adapters_add(launch=1, ws=P, ws_bytes=2**20)[0] == QMM_NO_ROOM
    assert adapters_add(rows=3000, launch=1)[0] == QMM_WORKSPACE_TOO_SMALL


def test_reference_step_by_hand():
    tables, lens, free = [[5, 3, -1], [0, -1, -1], [-1, -1, -1]], [20, 16, 0], [7, 6, 2]
    # 0 is cut by 5 to 15 (page 3 back), takes 2 (page 3 again); 1 takes 1 (page 2); 2 takes 33 of three pages: short
    out = ref.step(tables, lens, free, 16, 40, new=[2, 1, 33], keep=[15, -1, -1])
    assert out[0] == [0, 2, 3, 36] and out[1] == [2, 1, 0]
    assert out[2] == [5 * 16 + 15, 3 * 16, 2 * 16] + [-1] * 37
    assert out[3] == [15, 16, 16] + [-1] * 37 and out[4] == [0, 0, 1] + [2] * 33 + [-1] * 4
    assert tables == [[5, 3, -1], [0, 2, -1], [-1] * 3] and lens == [17, 17, 0] and free == [7, 6]


def test_reference_kept_by_hand():
    x = torch.tensor([1.0, 3.0, math.nan, 3.0, 2.0, -math.inf])
    e = math.exp(-1)
    assert torch.allclose(ref.kept(x), torch.tensor([e * e, 1, 0, 1, e, 0], dtype=torch.float64), atol=1e-15)
    assert ref.kept(x, temperature=0.0).tolist() == [0, 1, 0, 0, 0, 0]
    assert ref.kept(x, top_k=1).tolist() == [0, 1, 0, 0, 0, 0]
    assert ref.kept(x, top_p=0.5).tolist() == [0, 1, 0, 1, 0, 0]  # one of them holds 1 / (2 + e + e^2) < 0.5
    assert ref.kept(x, top_p=0.0).tolist() == [0, 1, 0, 0, 0, 0]
    assert ref.kept(x, min_p=0.3).tolist() == pytest.approx([0, 1, 0, 1, e, 0])
    assert ref.kept(torch.full((3,), -math.inf)) is None
    assert ref.kept(torch.tensor([math.inf, 3.0, math.inf])).tolist() == [1, 0, 1]
    w = torch.tensor([0.0, 1.0, 0.0, 3.0, 0.0], dtype=torch.float64)
    assert [ref.token(w, u)[0] for u in (0.0, 0.2499, 0.25, 0.99, 1.0, 2.0, -1.0, math.nan)] == [1, 1, 3, 3, 3, 3, 1, 1]
    assert ref.token(w, 0.5)[1] == 0.75 and ref.token(None, 0.5) == (-1, 0.0)
