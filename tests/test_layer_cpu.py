"""The norm's, the cache's and the attention's C entries without a GPU: sizes,
what a call plans, and refusals before anything touches the device."""
import ctypes

import pytest

from swarmllm_amd import _lib
from swarmllm_amd._lib import QMM_OK, QMM_UNSUPPORTED, QMM_WORKSPACE_TOO_SMALL, X_BF16, X_F16, X_F32, Cache, lib

P = ctypes.c_void_p(4096)  # a 16-byte aligned address that is never read


def need():
    return ctypes.c_size_t(123)


def cache(pages=100, heads=8, hd=128, page=64, **change):
    c = Cache(4096, 4096, 4096, 4096, pages, heads, hd, page)
    for k, v in change.items():
        setattr(c, k, v)
    return c


def attend(c=None, n=None, launch=0, **change):
    a = dict(q=P, q_dtype=X_F16, q_stride=32 * 128, q_head=128, tokens=4, heads=32, starts=P, lens=P, tables=P,
             table_stride=50, seqs=2, max_q=2, max_kv=3000, scale=0.1, window=0, sinks=None, out=P, out_dtype=X_F16,
             out_stride=32 * 128, ws=None, ws_bytes=0)
    a.update(change)
    n = n if n is not None else need()
    c = c or cache()
    st = lib().qmm_attend(ctypes.byref(c), a["q"], a["q_dtype"], a["q_stride"], a["q_head"], a["tokens"], a["heads"],
                          a["starts"], a["lens"], a["tables"], a["table_stride"], a["seqs"], a["max_q"], a["max_kv"],
                          a["scale"], a["window"], a["sinks"], a["out"], a["out_dtype"], a["out_stride"], a["ws"],
                          a["ws_bytes"], ctypes.byref(n), launch, 0)
    return st, n.value


def test_plane_bytes():
    codes, scales = ctypes.c_size_t(), ctypes.c_size_t()
    fn = lib().qmm_cache_plane_bytes
    assert fn(100, 8, 128, 64, ctypes.byref(codes), ctypes.byref(scales)) == QMM_OK
    assert codes.value == 100 * 8 * 128 * 64 and scales.value == codes.value // 16
    assert fn(2**31 - 1, 65535, 256, 256, ctypes.byref(codes), ctypes.byref(scales)) == QMM_OK
    assert codes.value == (2**31 - 1) * 65535 * 256 * 256
    for pages, heads, hd, page in ((0, 8, 128, 64), (-1, 8, 128, 64), (2**31, 8, 128, 64), (4, 0, 128, 64),
                                   (4, 65536, 128, 64), (4, 8, 80, 64), (4, 8, 32, 64), (4, 8, 512, 64), (4, 8, 128, 8),
                                   (4, 8, 128, 48), (4, 8, 128, 512)):
        assert fn(pages, heads, hd, page, ctypes.byref(codes), ctypes.byref(scales)) == QMM_UNSUPPORTED
    assert fn(4, 8, 128, 64, None, ctypes.byref(scales)) == QMM_UNSUPPORTED


def test_attend_plans():
    # short contexts in one launch, long ones in parts of a workspace; nothing to do needs nothing
    assert attend(max_kv=512) == (QMM_OK, 0)
    long = attend(seqs=1, tokens=1, max_q=1, max_kv=3200)
    assert long[0] == QMM_OK and long[1] > 0 and long[1] % 4 == 0
    assert attend(seqs=1, tokens=1, max_q=1, max_kv=10**9) == long  # cut at the table's row
    assert attend(seqs=1, tokens=1, max_q=1, max_kv=3200, window=128) == (QMM_OK, 0)
    for nothing in (dict(tokens=0), dict(seqs=0), dict(max_q=0)):
        assert attend(**nothing) == (QMM_OK, 0)
        assert attend(launch=1, **nothing) == (QMM_OK, 0)
    # many sequences fill the CUs without parts
    assert attend(seqs=200, tokens=200, max_q=1, max_kv=3200) == (QMM_OK, 0)
    # a chunk's workspace grows neither with the sequences' data nor past what its blocks need
    chunk = attend(seqs=1, tokens=128, max_q=128, max_kv=3200)
    assert chunk[0] == QMM_OK and 0 < chunk[1] <= 64 * 8 * 512 * (128 + 2) * 4
    # too small a workspace is refused before anything is enqueued, and says what it wants
    assert attend(seqs=1, tokens=1, max_q=1, max_kv=3200, launch=1, ws=P, ws_bytes=long[1] - 1) == \
        (QMM_WORKSPACE_TOO_SMALL, long[1])
    assert attend(seqs=1, tokens=1, max_q=1, max_kv=3200, launch=1) == (QMM_WORKSPACE_TOO_SMALL, long[1])


def test_attend_refusals():
    bad = [dict(q_dtype=3), dict(out_dtype=-1), dict(heads=0), dict(heads=12), dict(tokens=-1), dict(seqs=-1),
           dict(seqs=65536), dict(max_q=-1), dict(max_q=2**31, tokens=2**32), dict(max_kv=-1), dict(table_stride=-1),
           dict(table_stride=2**40), dict(window=-1), dict(q_head=64), dict(q_stride=-1), dict(out_stride=100),
           dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e31),
           dict(tokens=2**30, max_q=2**30, seqs=1)]
    for change in bad:
        assert attend(**change)[0] == QMM_UNSUPPORTED, change
    for c in (cache(pages=0), cache(hd=80), cache(page=20), cache(heads=0), cache(k_codes=None), cache(v_scales=4097)):
        assert attend(c)[0] == QMM_UNSUPPORTED
    for null in ("q", "out", "starts", "lens", "tables"):
        assert attend(max_kv=512, launch=1, **{null: None})[0] == QMM_UNSUPPORTED
    c = cache()
    assert lib().qmm_attend(ctypes.byref(c), P, 0, 4096, 128, 4, 32, P, P, P, 50, 2, 2, 512, 0.1, 0, None, P, 0, 4096, None,
                            0, None, 0, 0) == QMM_UNSUPPORTED
    assert lib().qmm_attend(None, P, 0, 4096, 128, 4, 32, P, P, P, 50, 2, 2, 512, 0.1, 0, None, P, 0, 4096, None, 0,
                            ctypes.byref(need()), 0, 0) == QMM_UNSUPPORTED


def test_cache_write_and_read_refusals():
    L, c = lib(), cache()
    r = ctypes.byref(c)
    assert L.qmm_cache_write(r, None, 1024, 128, None, 1024, 128, X_F32, None, 0, 0) == QMM_OK  # no tokens
    assert L.qmm_cache_read(r, None, 0, None, None, X_F16, 0) == QMM_OK
    for bad in ((P, 1024, 128, P, 1024, 128, 7, P, 1), (P, 1024, 64, P, 1024, 128, X_F32, P, 1),
                (P, 1024, 128, P, 1024, 127, X_F32, P, 1), (P, -1, 128, P, 1024, 128, X_F32, P, 1),
                (P, 1024, 128, P, -1, 128, X_F32, P, 1), (P, 1024, 128, P, 1024, 128, X_F32, P, -1),
                (None, 1024, 128, P, 1024, 128, X_F32, P, 1), (P, 1024, 128, None, 1024, 128, X_F32, P, 1),
                (P, 1024, 128, P, 1024, 128, X_F32, None, 1)):
        assert L.qmm_cache_write(r, *bad, 0) == QMM_UNSUPPORTED
    for bad in ((P, 1, P, P, 5), (P, -1, P, P, X_F16), (None, 1, P, P, X_F16), (P, 1, None, P, X_F16),
                (P, 1, P, None, X_F16)):
        assert L.qmm_cache_read(r, *bad, 0) == QMM_UNSUPPORTED
    odd = cache(k_scales=4098)
    assert L.qmm_cache_read(ctypes.byref(odd), P, 1, P, P, X_F16, 0) == QMM_UNSUPPORTED
    assert L.qmm_cache_read(None, P, 1, P, P, X_F16, 0) == QMM_UNSUPPORTED


def norm(**change):
    a = dict(x=P, dtype=X_F32, xs=512, r=P, rs=512, w=P, eps=1e-5, h=P, hs=512, xq=P, layout=_lib.ACT_Q8K, y=None,
             ydt=X_F32, ys=512, k=512, rows=2)
    a.update(change)
    return lib().qmm_rms_norm_act(*a.values(), 0)


def test_norm_refusals():
    for bad in (dict(x=None), dict(w=None), dict(xq=None), dict(dtype=3), dict(k=0), dict(k=510), dict(k=500),
                dict(k=2**31), dict(rows=0), dict(xs=511), dict(rs=511), dict(hs=511), dict(eps=-1.0),
                dict(eps=float("nan")), dict(layout=2), dict(y=P, ydt=9), dict(y=P, ys=100),
                dict(k=96, layout=_lib.ACT_Q8K), dict(k=100, layout=_lib.ACT_Q8_0)):
        assert norm(**bad) == QMM_UNSUPPORTED, bad
    L = lib()
    for bad in ((None, 0, P, X_F16, 512, 1), (P, 2, P, X_F16, 512, 1), (P, 0, None, X_F16, 512, 1),
                (P, 0, P, 3, 512, 1), (P, 0, P, X_F16, 500, 1), (P, 1, P, X_BF16, 48, 1), (P, 0, P, X_F16, 512, 0)):
        assert L.qmm_dequantize_act(*bad, 0) == QMM_UNSUPPORTED


@pytest.mark.parametrize("t,k,n,rows", [(12, 4096, 4096, 1), (12, 4096, 4096, 77), (14, 14336, 4096, 512), (8, 4096, 4096, 9)])
def test_products_of_planes_plan_the_slots_alone(t, k, n, rows):
    """The workspace of qmm_forward without the activation it holds first."""
    L, a, b = lib(), need(), need()
    assert L.qmm_forward(t, None, None, k, None, n, None, 0, ctypes.byref(a), k, n, rows, 0, 0) == QMM_OK
    assert L.qmm_forward_act(t, None, None, None, n, None, 0, ctypes.byref(b), k, n, rows, 0, 0) == QMM_OK
    act = L.qmm_act_bytes(L.qmm_act_layout(t, rows), k, rows)
    slots = a.value - (act + 255) // 256 * 256 if a.value > act else 0
    assert b.value == slots
    assert L.qmm_forward_act(t, P, None, P, n, None, 0, ctypes.byref(b), k, n, rows, 1, 0) == QMM_UNSUPPORTED
    assert L.qmm_forward_act(t, None, P, P, n, None, 0, ctypes.byref(b), k, n, rows, 1, 0) == QMM_UNSUPPORTED
    assert L.qmm_forward_act(t, P, P, P, n - 1, None, 0, ctypes.byref(b), k, n, rows, 0, 0) == QMM_UNSUPPORTED
    assert L.qmm_forward_act(3, P, P, P, n, None, 0, ctypes.byref(b), k, n, rows, 0, 0) == QMM_UNSUPPORTED
    assert L.qmm_forward_glu_act(t, 5, P, P, P, P, n, None, 0, ctypes.byref(b), k, n, rows, 0, 0) == QMM_UNSUPPORTED
    assert L.qmm_forward_shared_act(t, 0, None, None, None, None, P, None, 0, ctypes.byref(b), k, rows, 0, 0) == QMM_UNSUPPORTED


def test_addresses_off_16_bytes_are_refused():
    """The planes of an activation and the partial results of a context are read and written 16 bytes at a time."""
    odd = ctypes.c_void_p(4096 + 8)
    assert norm(xq=odd) == QMM_UNSUPPORTED
    L, n = lib(), need()
    assert L.qmm_dequantize_act(odd, _lib.ACT_Q8K, P, X_F16, 512, 1, 0) == QMM_UNSUPPORTED
    assert L.qmm_forward_act(12, P, odd, P, 64, None, 0, ctypes.byref(n), 512, 64, 1, 0, 0) == QMM_UNSUPPORTED
    assert L.qmm_forward_glu_act(12, 0, P, P, odd, P, 64, None, 0, ctypes.byref(n), 512, 64, 1, 0, 0) == QMM_UNSUPPORTED
    one, w, d = (ctypes.c_int64 * 1)(64), (ctypes.c_void_p * 1)(4096), (ctypes.c_void_p * 1)(4096)
    assert L.qmm_forward_shared_act(12, 1, w, one, d, one, odd, None, 0, ctypes.byref(n), 512, 1, 0, 0) == QMM_UNSUPPORTED
    long = dict(seqs=1, tokens=1, max_q=1, max_kv=3200)
    want = attend(**long)[1]
    assert attend(launch=1, ws=odd, ws_bytes=want, **long) == (QMM_UNSUPPORTED, want)


def test_attend_takes_the_injected_fault():
    lib().qmm_fail_next_launch()
    assert attend(max_kv=512)[0] == QMM_OK  # a plan does not
    assert attend(max_kv=512, launch=1, q=None)[0] == _lib.QMM_NO_ROOM
    assert attend(max_kv=512, launch=1, q=None)[0] == QMM_UNSUPPORTED  # once


@pytest.mark.parametrize("heads,hd", [(64, 128), (8, 256), (40, 64)])
@pytest.mark.parametrize("max_kv", [2000, 8192, 32768])
def test_partial_results_stay_within_a_round_of_the_cus(heads, hd, max_kv):
    """However many blocks stand behind the last whole round, their parts are no more than a round holds: 512
    workgroups of 128 query rows, or twice 256 of 256 in equal shares, a row's sums and its two numbers each."""
    most = 2 * 256 * 256 * (hd + 2) * 4 + 256 * 16
    for new in (5, 33, 40, 130, 700):
        for seqs in (1, 2, 31, 32, 33, 51, 63, 64, 65, 66, 127, 128, 129, 192, 200, 256, 257, 1025, 8193):
            st, got = attend(cache(pages=10**6, hd=hd), seqs=seqs, tokens=seqs * new, max_q=new, heads=heads,
                             max_kv=max_kv, table_stride=512, q_stride=heads * hd, q_head=hd, out_stride=heads * hd)
            assert st == QMM_OK and got <= most, (seqs, new, got)


@pytest.mark.parametrize("shape", [dict(seqs=1, tokens=1, max_q=1), dict(seqs=1, tokens=512, max_q=512),
                                   dict(seqs=2, tokens=4000, max_q=2000), dict(seqs=16, tokens=16, max_q=1)])
def test_a_window_past_the_context_plans_as_none(shape):
    """The largest number is a caller's way to say "no window"."""
    for max_kv in (700, 3200):
        none = attend(max_kv=max_kv, **shape)
        assert none[0] == QMM_OK
        for window in (max_kv, 2**31, 2**62, 2**63 - 1):
            assert attend(max_kv=max_kv, window=window, **shape) == none


@pytest.mark.parametrize("t,k,n,rows", [(12, 4096, 4096, 1), (12, 14336, 4096, 77), (14, 14336, 4096, 100), (8, 4096, 4096, 9)])
def test_a_workspace_of_products_off_16_bytes_is_refused(t, k, n, rows):
    """The slots of a K split and the GLU's products lie at its start and go 16 bytes at a time."""
    L, size = lib(), need()
    one, w, d = (ctypes.c_int64 * 1)(n), (ctypes.c_void_p * 1)(4096), (ctypes.c_void_p * 1)(4096)
    for at in (4097, 4100, 4104):
        odd = ctypes.c_void_p(at)
        for launch in (0, 1):
            # (w and xq missing where the call would launch: nothing may reach the device here)
            x, wp = (None, None) if launch else (P, P)
            for room in (0, 2**40):
                assert L.qmm_forward_act(t, P, P, P, n, odd, room, ctypes.byref(size), k, n, rows, 0, 0) == QMM_UNSUPPORTED
                assert L.qmm_forward_act(t, wp, x, P, n, odd, room, ctypes.byref(size), k, n, rows, launch, 0) == QMM_UNSUPPORTED
                assert L.qmm_forward_shared_act(t, 1, w, one, d, one, x, odd, room, ctypes.byref(size), k, rows, launch, 0) == QMM_UNSUPPORTED
                assert L.qmm_forward_glu_act(t, 0, wp, wp, x, P, n, odd, room, ctypes.byref(size), k, n, rows, launch, 0) == QMM_UNSUPPORTED
    assert L.qmm_forward_act(t, P, P, P, n, P, 2**40, ctypes.byref(size), k, n, rows, 0, 0) == QMM_OK
    assert L.qmm_forward_glu_act(t, 0, P, P, P, P, n, P, 2**40, ctypes.byref(size), k, n, rows, 0, 0) == QMM_OK
    assert L.qmm_forward_shared_act(t, 1, w, one, d, one, P, P, 2**40, ctypes.byref(size), k, rows, 0, 0) == QMM_OK


def test_slots_stay_inside_the_table():
    """A position behind the last page would index past the table, on the device; one before the first wraps around."""
    from types import SimpleNamespace

    import torch

    from swarmllm_amd import KvCache

    kv, table = SimpleNamespace(page=16), torch.tensor([5, 0, -1, 9], dtype=torch.int32)
    assert KvCache.slots(kv, table, 14, 4).tolist() == [94, 95, 0, 1]
    assert KvCache.slots(kv, table, 0, 64).numel() == 64 and KvCache.slots(kv, table, 64, 0).numel() == 0
    assert (KvCache.slots(kv, table, 32, 16) < 0).all()  # no page: padding
    for t, start, count in ((table, 64, 1), (table, 60, 5), (table, -1, 2), (table, 0, -1), (table[:0], 0, 1),
                            (table.view(2, 2), 0, 4), (table, 2**40, 1)):
        with pytest.raises(ValueError):
            KvCache.slots(kv, t, start, count)


def test_calls_of_more_threads_than_a_launch_takes_are_refused():
    """Past 2^32 threads in x a grid wraps around without an error."""
    L, r = lib(), ctypes.byref(cache())
    for tokens in (2**29 + 1, 2**40):
        assert L.qmm_cache_write(r, None, 1024, 128, None, 1024, 128, X_F32, None, tokens, 0) == QMM_UNSUPPORTED
        assert L.qmm_cache_read(r, None, tokens, None, None, X_F16, 0) == QMM_UNSUPPORTED
    many = dict(heads=256, q_stride=256 * 128, out_stride=256 * 128, max_kv=512)
    assert attend(cache(heads=256), seqs=2**15, tokens=2**15, max_q=1, **many)[0] == QMM_UNSUPPORTED
    assert attend(cache(heads=256), seqs=2**15 - 1, tokens=2**15, max_q=1, **many)[0] == QMM_OK
