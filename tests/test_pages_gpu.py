"""PageTables.step against the plain implementation: every array it writes, over steps that add, cut and run short."""
import random

import pytest
import torch

import batch_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def state(rng, seqs, row, pool, page, most):
    """Sequences of random lengths over the pages of a shuffled pool."""
    order = list(range(pool))
    rng.shuffle(order)
    tables, lens = [], []
    for _ in range(seqs):
        n = min(rng.randint(0, most), row * page, len(order) * page)
        have = -(-n // page)
        tables.append(order[:have] + [-1] * (row - have))
        order = order[have:]
        lens.append(n)
    return tables, lens, order


def device_state(tables, lens, free, pool, row, page):
    from swarmllm_amd import PageTables

    t = i32(tables) if tables and row else torch.empty((len(tables), row), dtype=torch.int32, device=DEV)
    return PageTables(t, i32(lens), i32(free + [-7] * (pool - len(free))), i32([len(free)]), page)


def check(pages, got, want, tables, lens, free):
    names = ("q_starts", "taken", "slots", "positions", "seq")
    for name, g, w in zip(names, got, want):
        assert g.tolist() == w, name
    assert pages.lens.tolist() == lens
    assert pages.tables.tolist() == tables
    n = int(pages.free_count)
    assert pages.free[:n].tolist() == free
    return n


@pytest.mark.parametrize("seqs,row,pool,page,most,new,slack", [
    (0, 4, 5, 16, 0, 0, 3), (1, 1, 1, 16, 0, 16, 0), (1, 3, 2, 64, 70, 1, 0), (3, 0, 4, 16, 0, 2, 0), (2, 5, 0, 32, 0, 3, 1),
    (8, 66, 600, 64, 4000, 1, 0), (64, 20, 700, 32, 500, 5, 7), (65, 40, 300, 16, 200, 60, -50), (100, 9, 120, 128, 900, 200, 0),
    (48, 130, 3000, 32, 3000, 900, 11), (700, 30, 9000, 16, 200, 250, 0), (1025, 6, 4000, 16, 60, 5, 0),
    (4096, 5, 9000, 16, 40, 3, 100), (3000, 3, 9000, 256, 600, 40, -1000)])
def test_steps(seqs, row, pool, page, most, new, slack):
    rng = random.Random(seqs * 1000 + row)
    tables, lens, free = state(rng, seqs, row, pool, page, most)
    pages = device_state(tables, lens, free, pool, row, page)
    for turn in range(4):
        add = [rng.choice([0, 1, rng.randint(0, new), -3]) for _ in range(seqs)]
        cut = [rng.choice([-1, n, max(0, n - rng.randint(0, 40)), 0 if rng.random() < 0.3 else n, n + 5]) for n in lens]
        tokens = max(0, sum(max(0, n) for n in add) + slack)
        keep = None if turn == 2 else cut
        got = pages.step(i32(add), tokens, keep=None if keep is None else i32(keep))
        want = ref.step(tables, lens, free, page, tokens, add, keep)
        held = check(pages, got, want, tables, lens, free)
        used = [p for t in tables for p in t if p >= 0]
        assert len(used) + held == pool and sorted(used + free) == list(range(pool))
    # cut alone, and nothing at all
    got = pages.step(keep=i32([0] * seqs))
    want = ref.step(tables, lens, free, page, 0, None, [0] * seqs)
    assert check(pages, got, want, tables, lens, free) == pool
    check(pages, pages.step(), ref.step(tables, lens, free, page, 0), tables, lens, free)


def test_a_step_that_cuts_what_the_last_one_added_changes_nothing():
    rng = random.Random(5)
    tables, lens, free = state(rng, 30, 40, 900, 16, 300)
    pages = device_state(tables, lens, free, 900, 40, 16)
    keep, new = i32([max(0, n - 20) for n in lens]), i32([rng.randint(0, 90) for _ in lens])
    first = pages.step(new, 3000, keep=keep)
    before = [t.clone() for t in (pages.tables, pages.lens, pages.free_count)]
    for _ in range(3):
        again = pages.step(new, 3000, keep=keep)
        for a, b in zip(first, again):
            assert torch.equal(a, b)
        for a, b in zip(before, (pages.tables, pages.lens, pages.free_count)):
            assert torch.equal(a, b)


def test_alloc_and_attention_s_arguments():
    from swarmllm_amd import KvCache, PageTables

    pages, kv = PageTables.alloc(3, 4, 6, page=16), KvCache.alloc(6, 2, 64, page=16)
    rows = pages.step(i32([20, 0, 5]), 25)
    assert rows.slots.tolist() == list(range(20)) + [32, 33, 34, 35, 36]
    assert pages.tables.tolist() == [[0, 1, -1, -1], [-1] * 4, [2, -1, -1, -1]] and int(pages.free_count) == 3
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v, q = (torch.randn(25, h, 64, generator=g, device=DEV) for h in (2, 2, 4))
    kv.write(k, v, rows.slots)
    assert torch.equal(rows.slots[20:], kv.slots(pages.tables[2], 0, 5))
    a = kv.attend(q, rows.q_starts, pages.lens, pages.tables, max_q=20)
    # the first token of each sequence sees itself alone
    _, values = kv.read(rows.slots[[0, 20]], torch.float32)
    assert torch.allclose(a[[0, 20]], values.repeat_interleave(2, 1), atol=2e-3)


def test_arrays_that_make_no_sense_change_nothing_outside():
    from swarmllm_amd import PageTables

    rng = random.Random(9)
    seqs, row, pool, page, tokens = 70, 9, 50, 16, 500
    for turn in range(6):
        big = [torch.full((64 + n + 64,), 777, dtype=torch.int32, device=DEV) for n in (seqs * row, seqs, pool, 1)]
        parts = [b[64:-64] for b in big]
        wild = [-2**31, -1, 0, 1, 17, 143, 145, 10**6, 2**31 - 1]
        for p in parts:
            p.copy_(i32([rng.choice(wild) for _ in range(p.numel())]))
        pages = PageTables(parts[0].view(seqs, row), parts[1], parts[2], parts[3], page)
        rows = pages.step(i32([rng.choice(wild) for _ in range(seqs)]), tokens, keep=i32([rng.choice(wild) for _ in range(seqs)]))
        starts = rows.q_starts.tolist()
        assert starts[0] == 0 and sorted(starts) == starts and starts[-1] <= tokens
        assert all(0 <= n <= row * page for n in pages.lens.tolist()) and 0 <= int(pages.free_count) <= pool
        for b in big:
            assert (b[:64] == 777).all() and (b[-64:] == 777).all()


def test_captured_steps_follow_the_lengths_on_the_device():
    rng = random.Random(3)
    tables, lens, free = state(rng, 20, 30, 500, 16, 200)
    pages = device_state(tables, lens, free, 500, 30, 16)
    new = i32([1] * 20)
    start = [t.clone() for t in (pages.tables, pages.lens, pages.free, pages.free_count)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pages.step(new, 24)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = pages.step(new, 24)
    for t, s in zip((pages.tables, pages.lens, pages.free, pages.free_count), start):
        t.copy_(s)
    for turn in range(40):
        if turn % 7 == 3:
            new.copy_(i32([rng.randint(0, 3) if i % 2 else 1 for i in range(20)]))
        want = ref.step(tables, lens, free, 16, 24, new.tolist())
        graph.replay()
        check(pages, rows, want, tables, lens, free)


def test_refusals():
    from swarmllm_amd import PageTables

    ok = PageTables.alloc(4, 5, 6, page=16)
    for bad in (lambda: PageTables(ok.tables[0], ok.lens, ok.free, ok.free_count, 16),
                lambda: PageTables(ok.tables.long(), ok.lens, ok.free, ok.free_count, 16),
                lambda: PageTables(ok.tables.t(), ok.lens, ok.free, ok.free_count, 16),
                lambda: PageTables(ok.tables, ok.lens[:3], ok.free, ok.free_count, 16),
                lambda: PageTables(ok.tables, ok.lens, ok.free.cpu(), ok.free_count, 16),
                lambda: PageTables(ok.tables, ok.lens, ok.free, ok.free, 16),
                lambda: PageTables(ok.tables, ok.lens, ok.free, ok.free_count, 24),
                lambda: PageTables.alloc(4097, 1, 1), lambda: PageTables.alloc(1, 2**24 + 1, 1),
                lambda: ok.step(i32([1] * 3), 5), lambda: ok.step(i32([1] * 4).long(), 5),
                lambda: ok.step(i32([1] * 4), -1), lambda: ok.step(i32([1] * 4), 5, keep=i32([1] * 4).cpu())):
        with pytest.raises(ValueError):
            bad()


def test_large_page_numbers_and_arrays_not_wanted():
    import ctypes

    from swarmllm_amd import PageTables
    from swarmllm_amd._lib import lib

    base = 2 ** 31 - 1 - 40
    for tokens in (90, 5000):
        pages = PageTables.alloc(3, 10, 40, page=256)
        pages.free += base
        rows = pages.step(i32([300, 256, 20]), 576 + 20)
        want = [[base, base + 1], [base + 2], [base + 3]]
        assert [[p for p in t if p >= 0] for t in pages.tables.tolist()] == want
        assert rows.slots[[0, 299, 300, 575]].tolist() == [base * 256, (base + 1) * 256 + 43, (base + 2) * 256, (base + 3) * 256 + 19]
        # only what is wanted: no keep, no positions, no sequences
        new = i32([40, 30, 20])
        q, taken = torch.empty(4, dtype=torch.int32, device=DEV), torch.empty(3, dtype=torch.int32, device=DEV)
        slots = torch.full((tokens + 8,), -7, dtype=torch.int64, device=DEV)
        assert lib().qmm_pages_step(ctypes.byref(pages._c), None, new.data_ptr(), tokens, q.data_ptr(), taken.data_ptr(),
                                    slots.data_ptr(), None, None, torch.cuda.current_stream().cuda_stream) == 0
        assert q.tolist() == [0, 40, 70, 90] and taken.tolist() == [40, 30, 20] and pages.lens.tolist() == [340, 286, 40]
        got = slots.tolist()
        assert got[:40] == [(base + 1) * 256 + 44 + i for i in range(40)] and got[40:70] == [(base + 4) * 256 + i for i in range(30)]
        assert got[70:90] == [(base + 3) * 256 + 20 + i for i in range(20)] and got[90:] == [-1] * (tokens - 90) + [-7] * 8
    rows = pages.step()  # nothing wanted
    assert rows.q_starts.tolist() == [0] * 4 and rows.slots.numel() == 0 and pages.lens.tolist() == [340, 286, 40]
    rows = pages.step(tokens=7)
    assert rows.q_starts.tolist() == [0] * 4 and rows.slots.tolist() == rows.seq.tolist() == rows.positions.tolist() == [-1] * 7
