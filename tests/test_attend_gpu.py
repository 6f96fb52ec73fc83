"""Attention over the paged Q8_0 cache against 64 bits (layer_reference.attend64,
where the allowed error is derived): one new token, a few and prompt chunks,
every head dim, page and group, ragged batches, windows, sinks, rows that see
nothing, pages that are not there, and cache offsets past 32 bits."""
import pytest
import torch

from layer_reference import attend64, rounding
from swarmllm_amd import KvCache

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def filled(pages, heads, hd, page, seed, scale=0.02):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kv = KvCache.alloc(pages, heads, hd, page)
    for i in (0, 2):
        kv.planes[i].copy_((torch.randn(kv.planes[i].shape, generator=g, device="cuda") * 50).round().clamp(-127, 127))
        kv.planes[i + 1].copy_(scale * (0.5 + torch.rand(kv.planes[i + 1].shape, generator=g, device="cuda")))
    return kv, g


def batch(new, kvl, heads, kv_heads, hd, page, dtype, seed=0, spare=0, sinks=False):
    per = max(1, -(-max(kvl) // page)) + spare
    kv, g = filled(len(new) * per + 2, kv_heads, hd, page, seed)
    tables = torch.randperm(kv.pages, generator=g, device="cuda")[: len(new) * per].view(len(new), per).int()
    starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    lens = torch.tensor(kvl, dtype=torch.int32, device="cuda")
    q = (1.5 * torch.randn(sum(new), heads, hd, generator=g, device="cuda")).to(dtype)
    sk = torch.randn(heads, generator=g, device="cuda") if sinks else None
    return kv, q, starts, lens, tables, sk


def check(got, want, tol):
    err = (got.double() - want).abs()
    ok = err <= tol + rounding(got.dtype) * (want.abs() + tol) + 2.0**-25
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} off, the worst by {float((err - tol).max()):.3g} over {float(tol[~ok].max()):.3g}"


def run(new, kvl, heads, kv_heads, hd, page, dtype, window=0, sinks=False, scale=None, seed=0, spare=0):
    kv, q, starts, lens, tables, sk = batch(new, kvl, heads, kv_heads, hd, page, dtype, seed, spare, sinks)
    got = kv.attend(q, starts, lens, tables, max_q=max(new), window=window, sinks=sk, scale=scale)
    assert got.dtype == dtype
    check(got, *attend64(kv, q, starts, lens, tables, hd ** -0.5 if scale is None else scale, window, sk))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("hd,page", [(64, 16), (64, 64), (96, 32), (128, 64), (128, 16), (256, 128), (256, 32), (128, 256)])
@pytest.mark.parametrize("n", [1, 15, 64, 65, 333])
def test_one_token(dtype, hd, page, n):
    run([1], [n], 8, 2, hd, page, dtype, seed=n)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (5, 1), (32, 4), (16, 1), (40, 2)])
@pytest.mark.parametrize("new", [1, 2, 3])
def test_groups_of_heads(heads, kv_heads, new):
    """Up to 20 query heads a kv head, with a few new tokens: rows past one, two and four tiles of 16."""
    run([new, new], [new + 100, new], heads, kv_heads, 128, 32, F16, seed=heads)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("new,kvl", [([5], [5]), ([31], [700]), ([32], [32]), ([33], [100]), ([128], [129]),
                                     ([129], [1000]), ([300], [300])])
def test_chunks(hd, new, kvl):
    for dtype in (F16, BF16):
        run(new, kvl, 8, 2, hd, 64, dtype, seed=hd + new[0])


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, False), (0, True), (1, False), (50, True), (64, False), (1000, True)])
def test_ragged_batches(page, window, sinks):
    """Prompts, few-token and one-token sequences of one call, some without cached tokens before them."""
    run([70, 1, 0, 3, 40, 1], [200, 517, 30, 3, 333, 1], 6, 3, 64, page, F16, window=window, sinks=sinks, seed=page)
    run([1, 1, 1], [1000, 40, 517], 8, 1, 128, page, BF16, window=window, sinks=sinks, seed=page)


@pytest.mark.parametrize("new,n", [(1, 20000), (2, 9001), (40, 5000)])
def test_long_contexts_joined_from_parts(new, n):
    run([new], [n], 8, 1, 128, 64, F16, seed=n)
    run([new, 1], [n, 7], 4, 1, 64, 16, BF16, seed=n, sinks=True)


@pytest.mark.parametrize("hd,page", [(64, 16), (64, 64), (96, 128), (128, 32), (128, 64)])
@pytest.mark.parametrize("window", [0, 2100])
def test_chunks_of_several_rounds_of_the_cus(hd, page, window):
    """More blocks of 256 rows than CUs (64 kv heads, 5 blocks of each): the
    first blocks in parts, the others whole, and a one-token sequence beside."""
    run([1100], [2400], 64, 64, hd, page, F16, window=window, seed=hd)
    run([300, 1, 290], [2300, 2100, 2048], 16, 4, hd, page, BF16, window=window, seed=hd, sinks=True)


@pytest.mark.parametrize("new,n", [(65, 2047), (520, 2049), (100, 10000)])
def test_blocks_of_128_and_256_rows(new, n):
    """Both sides of the lines between the two (rows past 256, contexts past 2048)."""
    for heads, kv_heads in ((4, 1), (2, 1), (12, 4)):
        run([new], [n], heads, kv_heads, 128, 64, F16, seed=n)


def test_rows_that_see_nothing():
    """kv_len under the new tokens (the first rows stand before position 0), no cached positions at all, tables of no page."""
    for new, kvl in (([1, 4, 3], [0, 2, 0]), ([40, 33], [7, 0])):
        for sinks in (False, True):
            kv, q, starts, lens, tables, sk = batch(new, kvl, 4, 2, 64, 16, F16, seed=1, sinks=sinks)
            got = kv.attend(q, starts, lens, tables, max_q=max(new), sinks=sk)
            want, tol = attend64(kv, q, starts, lens, tables, 0.125, 0, sk)
            check(got, want, tol)
            assert (got[: new[0] - kvl[0]] == 0).all()
            bad = torch.full_like(tables, -1)
            bad[:, ::2] = kv.pages
            assert (kv.attend(q, starts, lens, bad, max_q=max(new), sinks=sk) == 0).all()


@pytest.mark.parametrize("new", [[1, 1], [5, 2], [60, 33]])
@pytest.mark.parametrize("page", [16, 64])
def test_pages_outside_the_cache_count_as_not_there(new, page):
    kv, q, starts, lens, tables, _ = batch(new, [300, 290], 4, 2, 64, page, F16, seed=4)
    tables[0, 1], tables[1, 0], tables[1, 2] = -1, kv.pages, 2**31 - 1
    got = kv.attend(q, starts, lens, tables, max_q=max(new))
    check(got, *attend64(kv, q, starts, lens, tables, 0.125))


@pytest.mark.parametrize("new", [[1, 1], [3, 20]])
def test_what_no_position_reaches_may_hold_anything(new):
    """NaN and infinite scales (and codes) past the sequences' positions and outside the window."""
    for window in (0, 40):
        kv, q, starts, lens, tables, _ = batch(new, [100, 205], 4, 2, 64, 64, F16, seed=5, spare=1)
        clean = kv.attend(q, starts, lens, tables, max_q=max(new), window=window)
        want, tol = attend64(kv, q, starts, lens, tables, 0.125, window)
        check(clean, want, tol)
        for b, n in enumerate((100, 205)):
            for p in range(tables.shape[1] * 64):
                first = n - new[b] - window + 1 if window else 0
                if p >= n or p < first:
                    page, at = int(tables[b, p // 64]), p % 64
                    bad = float("nan") if p % 2 else float("inf")
                    kv.planes[1][page, :, at] = bad
                    kv.planes[3][page, :, :, at] = bad
        got = kv.attend(q, starts, lens, tables, max_q=max(new), window=window)
        assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides_outputs_and_rows_behind_the_last_sequence(dtype):
    kv, q, starts, lens, tables, _ = batch([3, 1], [50, 60], 4, 2, 64, 16, dtype, seed=6)
    want, tol = attend64(kv, q, starts, lens, tables, 0.125)
    rows = torch.full((7, 4 * 64 + 2 * 2 * 64 + 3), 1e4, device="cuda").to(dtype)  # fused rows, padded, odd distance
    rows[:4, : 4 * 64] = q.flatten(1)
    for odt in (F16, BF16, F32):
        out = torch.full((7, 5, 64), 7.0, device="cuda", dtype=odt)
        view = out.flatten(1)[:, : 4 * 64].unflatten(1, (4, 64))
        got = kv.attend(rows[:, : 4 * 64].unflatten(1, (4, 64)), starts, lens, tables, max_q=3, out=view)
        assert got is view
        check(got[:4], want, tol)
        assert (out[4:] == 7).all() and (out[:, 4] == 7).all()
    # a bound above every sequence's changes no bits of a short context
    a = kv.attend(q, starts, lens, tables, max_q=3)
    assert torch.equal(a, kv.attend(q, starts, lens, tables, max_q=3, max_kv=64))
    # rows past max_q stay, positions past max_kv are cut
    out = torch.full((4, 4, 64), 7.0, device="cuda", dtype=dtype)
    kv.attend(q, starts, lens, tables, max_q=2, out=out)
    assert (out[2] == 7).all() and (out[3] != 7).any()
    cut = kv.attend(q, starts, lens, tables, max_q=3, max_kv=48)
    check(cut, *attend64(kv, q, starts, lens, tables, 0.125, max_kv=48))


def test_large_scores_and_one_hot_weights():
    """Scores of hundreds: the weights are one-hot, the running maximum moves far between tiles."""
    kv, q, starts, lens, tables, _ = batch([1, 2, 40], [700, 500, 600], 4, 2, 64, 64, F16, seed=7)
    for scale in (8.0, -8.0, 0.0):
        got = kv.attend(q, starts, lens, tables, max_q=40, scale=scale)
        want, tol = attend64(kv, q, starts, lens, tables, scale)
        assert torch.isfinite(got).all()
        if scale == 0.0:
            check(got, want, tol)
    # keys that grow along the sequence, scores exact in f16: the last position wins
    kv.planes[0].zero_()
    kv.planes[1].fill_(1.0)
    p = torch.arange(700, device="cuda")
    slots = tables[0].long()[p // 64] * 64 + p % 64
    kv.planes[0][slots // 64, :, slots % 64, 0] = (p // 8).to(torch.int8)[:, None]
    q1 = torch.zeros(1, 4, 64, device="cuda", dtype=F16)
    q1[..., 0] = 1.0
    got = kv.attend(q1, starts[:2], lens[:1], tables[:1], max_q=1, scale=64.0)
    v = kv.read(slots[p // 8 == 699 // 8], F32)[1].double().mean(0).repeat_interleave(2, 0)
    assert (got[0].double() - v).abs().max() <= 2 * 2.0**-11 * v.abs().max() + 2.0**-10


def test_sinks_of_the_extremes():
    kv, q, starts, lens, tables, _ = batch([1, 5], [90, 40], 2, 1, 64, 16, F16, seed=8)
    none = kv.attend(q, starts, lens, tables, max_q=5)
    low = kv.attend(q, starts, lens, tables, max_q=5, sinks=torch.tensor([float("-inf"), -3e38], device="cuda"))
    assert torch.equal(low, none)
    high = kv.attend(q, starts, lens, tables, max_q=5, sinks=torch.tensor([1e4, 88.0], device="cuda"))
    assert (high == 0).all() or high.abs().max() < 1e-3


@pytest.mark.parametrize("new", [1, 5, 70])
def test_offsets_past_32_bits(new):
    heads, hd, page = 8, 128, 64
    pages = 2**32 // (page * heads * hd) + 40
    kv = KvCache.alloc(pages, heads, hd, page)
    tables = torch.arange(pages - 1, pages - 6, -1, device="cuda", dtype=torch.int32).view(1, 5)
    tables[0, 1] = 2
    n = 300
    slots = kv.slots(tables[0], 0, n)
    k, v = (torch.randn(n, heads, hd, device="cuda") for _ in range(2))
    kv.write(k, v, slots)
    small = KvCache.alloc(5, heads, hd, page)
    st = torch.arange(5, device="cuda", dtype=torch.int32).view(1, 5)
    small.write(k, v, small.slots(st[0], 0, n))
    q = torch.randn(new, 16, hd, device="cuda").half()
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = kv.attend(q, starts, lens, tables, max_q=new)
    assert torch.equal(got, small.attend(q, starts, lens, st, max_q=new))
    check(got, *attend64(small, q, starts, lens, st, hd ** -0.5))


def test_malformed_device_bounds_stay_inside():
    """q_starts and kv_lens that no plan could make are cut to what is there."""
    kv, q, starts, lens, tables, _ = batch([4, 4], [60, 60], 4, 2, 64, 16, F16, seed=9)
    out = torch.full_like(q, 7.0)
    for s in ([0, 100, 50], [-5, 4, 2**31 - 1], [8, 0, 4]):
        kv.attend(q, torch.tensor(s, dtype=torch.int32, device="cuda"), lens, tables, max_q=4, out=out)
    kv.attend(q, starts, torch.tensor([-7, 2**31 - 1], dtype=torch.int32, device="cuda"), tables, max_q=4, out=out)
    assert (out[:4] == 0).all() and torch.isfinite(out[4:]).all()


def test_refusals():
    kv, q, starts, lens, tables, _ = batch([2, 1], [20, 20], 4, 2, 64, 16, F16, seed=10)
    bad = [dict(q=q[:, :3]), dict(q=q.double()), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q.cpu()),
           dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(q_starts=starts[:2]), dict(q_starts=starts.long()),
           dict(kv_lens=lens.long()), dict(kv_lens=lens.cpu()), dict(tables=tables.long()), dict(tables=tables[:1]),
           dict(tables=tables[0]), dict(tables=tables.t().contiguous().t()), dict(max_q=-1), dict(window=-1), dict(max_kv=-1),
           dict(sinks=torch.zeros(3, device="cuda")), dict(sinks=torch.zeros(4, device="cuda").half()),
           dict(out=torch.empty(2, 4, 64, device="cuda").half()), dict(out_dtype=torch.float64),
           dict(out=torch.empty(3, 4, 128, device="cuda").half()[..., :64])]
    base = dict(q=q, q_starts=starts, kv_lens=lens, tables=tables, max_q=2)
    for change in bad:
        with pytest.raises(ValueError):
            kv.attend(**{**base, **change})
    assert kv.attend(q[:0], starts[:1] * 0, lens[:0], tables[:0], max_q=0).shape == (0, 4, 64)
    out = torch.full_like(q, 3.0)
    assert (kv.attend(q, starts[:1], lens[:0], tables[:0], max_q=2, out=out) == 3).all()


@pytest.mark.parametrize("new,most", [(5, 3), (40, 7), (300, 40), (600, 290)])
def test_rows_past_max_q_are_left_and_move_no_other(new, most):
    """Positions go by q_starts and kv_lens alone: the rows inside max_q are those of a call that has them all."""
    kv, q, starts, lens, tables, _ = batch([new, 1], [new + 900, 300], 8, 2, 64, 32, F16, seed=new)
    want, tol = attend64(kv, q, starts, lens, tables, 0.125)
    out = torch.full_like(q, 7.0)
    kv.attend(q, starts, lens, tables, max_q=most, out=out)
    inside = torch.arange(new + 1, device="cuda")
    inside = (inside < most) | (inside == new)
    check(out[inside], want[inside], tol[inside])
    assert (out[~inside] == 7).all()


@pytest.mark.parametrize("hd,page,dtype", [(64, 16, F16), (64, 64, BF16), (96, 32, BF16), (128, 64, F16), (128, 16, BF16)])
@pytest.mark.parametrize("window,sinks", [(0, False), (0, True), (2100, False)])
def test_blocks_in_equal_shares(hd, page, dtype, window, sinks):
    """480 blocks of 256 rows by the longest sequence, 200 and some in fact: chunks, a prompt without a past, one
    whose first rows stand before the cache, a few-token and an absent sequence, whole tables' pages apart."""
    run([1100, 1, 700, 0, 300, 430], [2300, 2100, 700, 40, 2600, 200], 20, 20, hd, page, dtype, window=window,
        sinks=sinks, seed=hd + page)


@pytest.mark.parametrize("heads,kv_heads", [(12, 4), (40, 8), (24, 2)])
def test_shares_of_shared_heads(heads, kv_heads):
    """Groups of 3, 5 and 12: blocks that end inside a token's heads."""
    new = [2100, 900, 1500] if kv_heads == 2 else [1500, 2000, 40, 1000] * (2 if kv_heads == 4 else 1)
    kvl = [n + 100 * i for i, n in enumerate(new)]
    kvl[0] += 1500
    run(new, kvl, heads, kv_heads, 64, 64, F16, seed=heads)


def test_more_sequences_than_threads_beside_a_prompt():
    """A search of several rounds: prompts among 700 sequences of one token, and of none."""
    new, kvl = [1] * 700, [1 + i % 70 for i in range(700)]
    for i, (n, k) in {3: (500, 2200), 511: (300, 300), 512: (290, 2000), 600: (0, 9), 699: (512, 2100)}.items():
        new[i], kvl[i] = n, k
    per = 2200 // 256 + 1
    kv, g = filled(per * 5 + 700, 1, 64, 256, 3)
    tables = torch.full((700, per), -1, dtype=torch.int32, device="cuda")
    tables[:, 0] = torch.arange(700, dtype=torch.int32, device="cuda")
    for x, i in enumerate((3, 511, 512, 600, 699)):
        tables[i] = torch.arange(700 + x * per, 700 + (x + 1) * per, dtype=torch.int32, device="cuda")
    starts = torch.tensor([sum(new[:b]) for b in range(701)], dtype=torch.int32, device="cuda")
    lens = torch.tensor(kvl, dtype=torch.int32, device="cuda")
    q = (1.5 * torch.randn(sum(new), 1, 64, generator=g, device="cuda")).half()
    got = kv.attend(q, starts, lens, tables, max_q=512)
    check(got, *attend64(kv, q, starts, lens, tables, 0.125))
