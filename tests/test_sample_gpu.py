"""sample against the definition in 64 bits. The tokens have to be equal; where the number falls within 2^-40 of the
total weight of a border between two of them, either one is right (sums in 64 bits are off by 2^-52 a term)."""
import math

import pytest
import torch

import batch_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = math.inf, math.nan


def logits(seed, rows, vocab, spread=2.2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g, device=DEV)
    few = torch.randint(vocab, (rows, min(vocab, 50)), generator=g, device=DEV)
    return x.scatter_add_(1, few, 7.0 + 3.0 * torch.randn(few.shape, generator=g, device=DEV))


def vec(v, dtype=torch.float32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def check(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    import swarmllm_amd as sa

    t = {n: None if v is None else vec(v, torch.int32 if n == "top_k" else torch.float32)
         for n, v in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p))}
    u = vec(u)
    out = sa.sample(x, u, **t)
    ids, probs = out.ids.tolist(), out.probs.tolist()
    f = {n: v.tolist() if v is not None else None for n, v in t.items()}
    for r, number in enumerate(u.tolist()):
        w = ref.kept(x[r].float(), *(f[n][r] if f[n] is not None else off
                                     for n, off in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))))
        want, p = ref.token(w, number)
        what = (r, number, {n: v[r] for n, v in f.items() if v is not None})
        if ids[r] != want:
            assert want >= 0 and 0 <= ids[r] < x.shape[1] and w[ids[r]] > 0, (ids[r], want, what)
            sums = w.cumsum(0)
            off = min(abs(number * sums[-1] - sums[ids[r]]), abs(number * sums[-1] - sums[ids[r]] + w[ids[r]]))
            assert off < 2.0 ** -40 * sums[-1], (ids[r], want, what)
            p = float(w[ids[r]] / sums[-1])
        # one rounding to f32 (2^-24 of the value, and 2^-150, half its least step, below its normal range), and 64-bit sums
        assert abs(probs[r] - p) <= 2.0 ** -23 * p + 2.0 ** -149, (probs[r], p, what)
    return out


SIZES = [1, 2, 3, 63, 64, 255, 257, 1023, 1024, 1025, 4097, 50257, 128256, 262147, 524288]


@pytest.mark.parametrize("vocab", SIZES)
def test_whole_rows(vocab):
    rows = 6 if vocab > 10000 else 40
    x = logits(vocab, rows, vocab)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(vocab)).tolist()
    u[:4] = [0.0, 1.0 - 2.0 ** -24, 1.0, 0.5]
    check(x, u)
    check(x, u, temperature=[0.3 + 0.3 * r for r in range(rows)])
    check(x, u, temperature=[0.0] * rows)


@pytest.mark.parametrize("vocab", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_settings(vocab, dtype):
    rows = 12 if vocab > 10000 else 40
    x = logits(vocab + 1, rows, vocab).to(dtype)
    g = torch.Generator().manual_seed(vocab)
    u = torch.rand(rows, generator=g).tolist()
    temperature = (0.4 + 1.4 * torch.rand(rows, generator=g)).tolist()
    temperature[1] = 0.0
    k = [(1, 0, 40, 5, 100, 700, 1024, 1025, 3000, 40000)[r % 10] for r in range(rows)]
    p = [(0.9, 0.5, 1.0, 0.99, 0.0, 0.9999)[r % 6] for r in range(rows)]
    m = [(0.0, 0.1, 0.0, 0.003, 1.0)[r % 5] for r in range(rows)]
    for settings in (dict(top_k=k), dict(top_p=p), dict(min_p=m), dict(top_k=k, top_p=p), dict(top_k=k, min_p=m),
                     dict(top_p=p, min_p=m), dict(top_k=k, top_p=p, min_p=m)):
        check(x, u, temperature=temperature, **settings)
    check(x, u, top_p=p)


@pytest.mark.parametrize("vocab", [1, 5, 1000, 3333, 40000, 524288])
def test_equal_logits(vocab):
    # one value alone, two values, and values of few bits: many places at every border
    flat = torch.full((1, vocab), -3.25, device=DEV)
    two = flat.clone()
    two[0, vocab // 3:: 3] = -3.0
    few = (logits(3, 1, vocab) / 2).round()
    x = torch.cat([flat, two, few]).repeat_interleave(7, 0)
    k = [1, 2, vocab // 2, vocab - 1, 1500, 0, 1024] * 3
    p = [1.0, 0.5, 0.7, 0.999, 1e-6, 0.3, 1.0] * 3
    for u in (0.0, 0.123, 0.77, 1.0 - 2.0 ** -24):
        check(x, [u] * 21, top_k=k)
        check(x, [u] * 21, top_p=p)
        check(x, [u] * 21, top_k=k, top_p=p, min_p=[0.0, 0.5, 0.9] * 7)


def test_every_number_draws_its_token():
    x = vec([[0.0, 1.0, -INF, 1.0, 0.5, -2.0, NAN]]).repeat(4096, 1)
    u = [i / 4096 for i in range(4096)]
    out = check(x, u)
    got = torch.bincount(out.ids.long(), minlength=7).double() / 4096
    w = ref.kept(x[0])
    assert (got - w / w.sum()).abs().max() <= 1 / 4096
    check(x, u, top_k=[3] * 4096)
    check(x, u, top_p=[0.6] * 4096)
    check(x, u, temperature=[2.0] * 4096, min_p=[0.5] * 4096)


@pytest.mark.parametrize("vocab", [9, 3000, 70000])
def test_masks_infinities_and_nan(vocab):
    x = logits(vocab, 9, vocab)
    x[0] = -INF
    x[1, :] = -INF
    x[1, vocab - 1] = 2.0
    x[2, : vocab // 2] = NAN
    x[3, 1] = x[3, vocab - 2] = INF
    x[4] = torch.finfo(torch.float32).min
    x[4, 3] = 0.0
    x[5] = NAN
    x[6] = torch.finfo(torch.float32).min
    x[7, ::2] = torch.finfo(torch.float32).max
    x[8] *= 1e30
    for u in (0.0, 0.4, 1.0 - 2.0 ** -24, 1.0, 3.0, -1.0, NAN):
        for settings in (dict(), dict(top_k=[2] * 9), dict(top_p=[0.8] * 9), dict(min_p=[0.2] * 9),
                         dict(top_k=[5000] * 9, top_p=[0.9] * 9), dict(temperature=[0.0] * 9)):
            check(x, [u] * 9, **settings)


def test_settings_past_their_range():
    x = logits(1, 12, 5000)
    u = [0.3, 0.9] * 6
    check(x, u, temperature=[NAN, -1.0, INF, 1e-38, 1e-45, 1e30, 3e38, -0.0, 1e-6, 50.0, 1.0, -INF])
    check(x, u, temperature=[NAN, -1.0, INF, 1e-38, 1e-45, 1e30, 3e38, -0.0, 1e-6, 50.0, 1.0, -INF], top_k=[70, 2000] * 6,
          top_p=[0.9, 0.5, 1.0] * 4)
    wild = [NAN, -1.0, INF, 1e-38, 1e-45, 1e30, 3e38, -0.0, 1e-6, 50.0, 1.0, -INF]
    check(x, u, temperature=wild, top_p=[0.9, 0.5, 0.3] * 4)
    check(x, u, temperature=wild, top_k=[3000] * 12)
    huge = x.clone()
    huge[:, ::3] = torch.finfo(torch.float32).max
    huge[:, 1::3] = torch.finfo(torch.float32).min
    check(huge, u, temperature=wild, top_p=[0.9, 0.5, 0.3] * 4)
    check(huge, u, temperature=wild, top_k=[3000] * 12)
    check(x, u, top_k=[-2**31, -1, 0, 1, 4999, 5000, 5001, 2**31 - 1, 2, 1024, 1025, 4096])
    check(x, u, top_p=[NAN, -1.0, 0.0, 1e-30, 1.0, 2.0, INF, -INF, 1.0 - 2.0 ** -24, 0.5, 1e-3, 0.999])
    check(x, u, min_p=[NAN, -1.0, 0.0, 1e-30, 1.0, 2.0, INF, -INF, 1.0 - 2.0 ** -24, 0.5, 1e-3, 1e-45])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_row_does_not_depend_on_its_place(dtype):
    import swarmllm_amd as sa

    x = logits(2, 40, 5004).to(dtype)
    g = torch.Generator(device=DEV).manual_seed(2)
    u, t, p = (torch.rand(40, generator=g, device=DEV) for _ in range(3))
    k = torch.randint(0, 3000, (40,), generator=g, device=DEV).to(torch.int32)
    want = sa.sample(x, u, temperature=t, top_k=k, top_p=p)
    whole = sa.sample(x, u)
    wide = torch.full((40, 5100), 99.0, device=DEV, dtype=dtype)
    for off in (1, 2, 3, 4, 8):
        view = wide[:, off:off + 5004]
        view.copy_(x)
        for got, right in ((sa.sample(view, u, temperature=t, top_k=k, top_p=p), want), (sa.sample(view, u), whole)):
            assert torch.equal(got.ids, right.ids) and torch.equal(got.probs, right.probs)
        wide.fill_(99.0)
    for r in (0, 17, 39):
        s = slice(r, r + 1)
        got = sa.sample(x[s], u[s], temperature=t[s], top_k=k[s], top_p=p[s])
        assert torch.equal(got.ids, want.ids[s]) and torch.equal(got.probs, want.probs[s])
        got = sa.sample(x[s], u[s])
        assert torch.equal(got.ids, whole.ids[s]) and torch.equal(got.probs, whole.probs[s])


def test_many_rows():
    # more rows than a launch takes: every row as on its own
    import swarmllm_amd as sa

    few = logits(6, 25, 1300)
    x = few.repeat(200, 1)
    g = torch.Generator(device=DEV).manual_seed(6)
    u, t, p, m = (torch.rand(25, generator=g, device=DEV) for _ in range(4))
    k = torch.randint(0, 1300, (25,), generator=g, device=DEV).to(torch.int32)
    for settings in ((t, None, None, None), (t, None, p, None), (t, k, p, m * 0.1)):
        want = sa.sample(few, u, *settings)
        got = sa.sample(x, u.repeat(200), *(None if v is None else v.repeat(200) for v in settings))
        assert torch.equal(got.ids.view(200, 25), want.ids.expand(200, 25))
        assert torch.equal(got.probs.view(200, 25), want.probs.expand(200, 25))


def test_captured_and_on_another_stream():
    import swarmllm_amd as sa

    x = logits(4, 8, 20000)
    g = torch.Generator(device=DEV).manual_seed(4)
    u, t = (torch.rand(8, generator=g, device=DEV) for _ in range(2))
    k = vec([0, 50, 2000, 1, 0, 9, 5000, 30], torch.int32)
    p = vec([0.9, 0.9, 0.8, 1.0, 1.0, 0.5, 0.99, 0.0])
    want = sa.sample(x, u, t, k, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sa.sample(x, u, t, k, p)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.ids, want.ids) and torch.equal(got.probs, want.probs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sa.sample(x, u, t, k, p)
    for turn in range(4):
        x.mul_(0.9)
        u.copy_(u.roll(1))
        graph.replay()
        want = sa.sample(x, u, t, k, p)
        assert torch.equal(out.ids, want.ids) and torch.equal(out.probs, want.probs)
        check(x, u.tolist(), t.tolist(), k.tolist(), p.tolist())


def test_refusals():
    import swarmllm_amd as sa

    x, u = torch.randn(3, 100, device=DEV), torch.rand(3, device=DEV)
    assert sa.sample(x[:0], u[:0]).ids.shape == (0,)
    for bad in (lambda: sa.sample(x[0], u), lambda: sa.sample(x.double(), u), lambda: sa.sample(x.cpu(), u),
                lambda: sa.sample(x.t(), u), lambda: sa.sample(x, u[:2]), lambda: sa.sample(x, u.double()),
                lambda: sa.sample(x, u.cpu()), lambda: sa.sample(x, None), lambda: sa.sample(x, u, temperature=u[:2]),
                lambda: sa.sample(x, u, top_k=u), lambda: sa.sample(x, u, top_p=u.long()), lambda: sa.sample(x[:, :0], u),
                lambda: sa.sample(torch.empty(3, 2 ** 19 + 1, device=DEV), u)):
        with pytest.raises(ValueError):
            bad()


def test_rows_far_apart():
    import swarmllm_amd as sa

    x = logits(11, 4, 20011).bfloat16()
    step = 2 ** 30 + 3
    far = torch.empty(3 * step + 20011, dtype=torch.bfloat16, device=DEV).as_strided((4, 20011), (step, 1))
    far.copy_(x)
    u = vec([0.1, 0.5, 0.9, 0.99])
    k, p = vec([0, 30, 5000, 0], torch.int32), vec([0.9, 1.0, 0.99, 0.5])
    for settings in ((None, None, None), (None, k, None), (None, None, p), (u, k, p)):
        got, want = sa.sample(far, u, *settings), sa.sample(x, u, *settings)
        assert torch.equal(got.ids, want.ids) and torch.equal(got.probs, want.probs)


def test_two_calls_at_once():
    import swarmllm_amd as sa

    sets = []
    for rows, vocab in ((40, 30000), (3, 128256), (300, 5000)):
        x = logits(rows, rows, vocab)
        g = torch.Generator(device=DEV).manual_seed(rows)
        u, t = (torch.rand(rows, generator=g, device=DEV) for _ in range(2))
        k = torch.randint(0, 900, (rows,), generator=g, device=DEV).to(torch.int32)
        sets.append((x, u, t, k * (k % 3 == 0), 0.9 * torch.ones_like(u)))
    want = [sa.sample(*s) for s in sets]
    streams, outs = [torch.cuda.Stream() for _ in sets], [[] for _ in sets]
    torch.cuda.synchronize()
    for turn in range(5):
        for stream, s, out in zip(streams, sets, outs):
            with torch.cuda.stream(stream):
                out.append(sa.sample(*s))
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert all(torch.equal(o.ids, w.ids) and torch.equal(o.probs, w.probs) for o in out)


def test_without_chances():
    import ctypes

    import swarmllm_amd as sa
    from swarmllm_amd._lib import X_F32, lib

    x, u = logits(12, 9, 9000), vec([0.05 + 0.1 * i for i in range(9)])
    t, k, p = vec([1.0, 0.0, 0.5] * 3), vec([0, 0, 0, 5, 80, 2000, 0, 0, 1], torch.int32), vec([0.9, 0.9, 1.0] * 3)
    for settings in ((None, None, None), (t, None, None), (t, k, p)):
        want = sa.sample(x, u, *settings).ids
        ids, need = torch.full((9,), -7, dtype=torch.int32, device=DEV), ctypes.c_size_t()
        ptrs = [None if v is None else v.data_ptr() for v in settings] + [None]
        call = lambda ws, size, launch: lib().qmm_sample(x.data_ptr(), X_F32, 9000, u.data_ptr(), *ptrs, ids.data_ptr(), None, 9000,
                                                         9, ws, size, ctypes.byref(need), launch,
                                                         torch.cuda.current_stream().cuda_stream)
        assert call(None, 0, 0) == 0
        ws = torch.empty(need.value, dtype=torch.uint8, device=DEV)
        assert call(ws.data_ptr(), need.value, 1) == 0
        assert torch.equal(ids, want)
