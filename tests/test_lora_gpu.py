"""Adapters.add against the sums in 64 bits."""
import pytest
import torch

import batch_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(seed, rows, k, n, rank, slots, x="f32", w="bf16", order="mixed"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    xs = torch.randn(rows, k, generator=g, device=DEV)
    xs[:, :: max(1, k // 7)] *= 20.0
    a = (torch.randn(slots, rank, k, generator=g, device=DEV) / k ** 0.5).to(T[w])
    b = (0.1 * torch.randn(slots, n, rank, generator=g, device=DEV)).to(T[w])
    scales = torch.rand(slots, generator=g, device=DEV) + 0.5
    ids = torch.randint(-1, slots, (rows,), generator=g, device=DEV).to(torch.int32)
    if order == "runs":
        ids = ids.sort().values.contiguous()
    if order == "one":
        ids.fill_(slots - 1)
    y = torch.randn(rows, n, generator=g, device=DEV)
    return xs.to(T[x]), a, b, scales, ids, y


def close(got, want, bound):
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() - bound).max())


CASES = [(1, 32, 1, 8, 1, "one"), (1, 4096, 4096, 16, 4, "one"), (2, 64, 17, 8, 3, "mixed"), (5, 96, 63, 24, 2, "mixed"),
         (16, 512, 65, 16, 16, "mixed"), (17, 544, 129, 40, 5, "mixed"), (21, 4096, 1024, 16, 24, "mixed"),
         (33, 14336, 257, 64, 4, "runs"), (64, 2880, 300, 128, 40, "mixed"), (65, 1024, 1000, 16, 70, "mixed"),
         (77, 4096, 513, 32, 3, "runs"), (200, 8192, 96, 56, 2, "runs"), (513, 256, 777, 64, 6, "runs"),
         (1000, 320, 64, 8, 100, "mixed"), (1300, 64, 3, 128, 2, "mixed"),
         (70, 1024, 1000, 64, 70, "mixed"), (300, 4096, 513, 16, 7, "mixed"), (300, 1024, 2100, 8, 40, "mixed"),
         (1025, 32, 1, 8, 1, "one"), (1030, 96, 63, 24, 2, "mixed"), (1100, 544, 129, 40, 5, "mixed"),
         (2100, 4096, 513, 16, 24, "mixed"), (1500, 256, 777, 64, 70, "mixed"), (1040, 320, 64, 8, 1100, "mixed"),
         (64, 14336, 2100, 128, 40, "mixed"), (20, 8192, 40000, 128, 3, "mixed"), (9, 28672, 8192, 128, 2, "runs"),
         (70, 8192, 8192, 96, 70, "mixed")]


@pytest.mark.parametrize("x,w", [("f32", "bf16"), ("f32", "f16"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"),
                                 ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("rows,k,n,rank,slots,order", CASES)
def test_against_64_bits(rows, k, n, rank, slots, order, x, w):
    from swarmllm_amd import Adapters

    xs, a, b, scales, ids, y = make(rows + k, rows, k, n, rank, slots, x, w, order)
    want, bound = ref.adapters(y, xs, ids, a, b, scales)
    out = torch.full_like(y, float("nan"))
    got = Adapters(a, b, scales).add(y, xs, ids, out=out)
    assert got is out
    close(got, want, bound)
    none = ids < 0
    assert torch.equal(got[none], y[none])
    inplace = y.clone()
    assert Adapters(a, b, scales).add(inplace, xs, ids) is inplace
    assert torch.equal(inplace, got)


@pytest.mark.parametrize("w", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,n,rank,slots,order", CASES)
def test_whole_numbers_come_out_whole(rows, k, n, rank, slots, order, w):
    # every product and sum is a whole number below 2^24, and x's take more bits than 16-bit types hold
    from swarmllm_amd import Adapters

    xs, a, b, _, ids, y = make(rows + 7 * k, rows, k, n, rank, slots, "f32", w, order)
    g = torch.Generator(device=DEV).manual_seed(rows)
    xs = torch.zeros_like(xs)
    for _ in range(8):  # eight places of each row
        at = torch.randint(k, (rows, 1), generator=g, device=DEV)
        xs.scatter_(1, at, torch.randint(-4095, 4096, (rows, 1), generator=g, device=DEV).float())
    a = torch.randint(-2, 3, a.shape, generator=g, device=DEV).to(T[w])
    b = torch.randint(-1, 2, b.shape, generator=g, device=DEV).to(T[w])
    y = torch.randint(-1000, 1000, y.shape, generator=g, device=DEV).float()
    want, _ = ref.adapters(y, xs, ids, a, b, None)
    assert want.abs().max() < 2 ** 24
    assert torch.equal(Adapters(a, b).add(y.clone(), xs, ids).double(), want)


@pytest.mark.parametrize("rows", [1, 21, 100, 300, 1100])
def test_shared_projections_equal_their_own(rows):
    from swarmllm_amd import Adapters

    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(rows, 1024, generator=g, device=DEV)
    ids = torch.randint(-1, 6, (rows,), generator=g, device=DEV).to(torch.int32)
    ads, ys = [], []
    for n, rank in ((1024, 16), (130, 16), (256, 8), (77, 64)):
        a, b = torch.randn(6, rank, 1024, generator=g, device=DEV) / 32, torch.randn(6, n, rank, generator=g, device=DEV)
        ads.append(Adapters(a.bfloat16(), b.bfloat16(), torch.rand(6, generator=g, device=DEV)))
        ys.append(torch.randn(rows, n, generator=g, device=DEV))
    for count in (1, 2, 3, 4):
        outs = [torch.empty_like(y) for y in ys[:count]]
        got = Adapters.add_shared(ys[:count], x, ads[:count], ids, outs=outs)
        for y, ad, o in zip(ys, ads, got):
            want, bound = ref.adapters(y, x, ids, ad.a, ad.b, ad.scales)
            close(o, want, bound)


def test_strides_alignment_and_what_lies_between():
    from swarmllm_amd import Adapters

    for rows in (3, 40, 270, 1050, 90):
        xs, a, b, scales, ids, y = make(rows, rows, 256, 50, 16, 3)
        wide = torch.full((rows, 400), 5.0, device=DEV)
        for off in (0, 1, 4):
            xv = torch.zeros(rows, 300, device=DEV)[:, off:off + 256]
            xv.copy_(xs)
            view = wide[:, 30 + off:80 + off]
            view.copy_(y)
            want, bound = ref.adapters(y, xs, ids, a, b, scales)
            Adapters(a, b, scales).add(view, xv, ids)
            close(view, want, bound)
            view.fill_(5.0)
            assert (wide == 5.0).all()
    # leading dimensions
    got = Adapters(a, b, scales).add(y.view(9, 10, 50).clone(), xs.view(9, 10, 256), ids)
    assert got.shape == (9, 10, 50)
    close(got.view(90, 50), want, bound)


@pytest.mark.parametrize("rows", [16, 70, 300, 1100])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_an_adapter_reaches_its_own_rows_only(rows, bad):
    from swarmllm_amd import Adapters

    xs, a, b, scales, ids, y = make(rows, rows, 512, 100, 16, 4)
    ids = (torch.arange(rows, device=DEV) % 5).to(torch.int32)  # 4 names no slot
    want, bound = ref.adapters(y, xs, ids, a, b, scales)
    a[2], b[1, :, 3], xs[3], scales[3] = bad, bad, bad, bad
    got = Adapters(a, b, scales).add(y.clone(), xs, ids)
    mine = (ids == 0) | (ids == 4)
    mine[3] = False
    close(got[mine], want[mine], bound[mine])
    assert not got[ids == 2].isfinite().any()
    assert not got[ids == 1].isfinite().any()


def test_ids_outside_the_slots_and_no_slots():
    from swarmllm_amd import Adapters

    xs, a, b, scales, ids, y = make(1, 40, 64, 30, 8, 3)
    ids.copy_(torch.tensor([-2**31, -1, 3, 2**31 - 1] * 10, dtype=torch.int32))
    out = torch.empty_like(y)
    assert torch.equal(Adapters(a, b, scales).add(y, xs, ids, out=out), y)
    empty = Adapters(a[:0], b[:0], scales[:0])
    assert torch.equal(empty.add(y.clone(), xs, ids.fill_(0)), y)
    assert Adapters(a, b).add(y[:0], xs[:0], ids[:0]).shape == (0, 30)


@pytest.mark.parametrize("rows", [4, 120, 300, 1100])
def test_captured_and_on_another_stream(rows):
    from swarmllm_amd import Adapters

    xs, a, b, scales, ids, y = make(rows, rows, 1024, 500, 16, 6)
    ad, out = Adapters(a, b, scales), torch.empty_like(y)
    want = ad.add(y.clone(), xs, ids)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ad.add(y.clone(), xs, ids)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ad.add(y, xs, ids, out=out)
    for turn in range(4):
        ids.copy_(ids.roll(1))
        xs.mul_(0.5)
        graph.replay()
        want, bound = ref.adapters(y, xs, ids, a, b, scales)
        close(out, want, bound)
        assert torch.equal(out, ad.add(y.clone(), xs, ids))


def test_refusals():
    from swarmllm_amd import Adapters

    xs, a, b, scales, ids, y = make(1, 10, 64, 30, 8, 3)
    ok = Adapters(a, b, scales)
    other, other_y = Adapters(a[:2].contiguous(), b[:2].contiguous()), y.clone()
    for bad in (lambda: Adapters(a[0], b), lambda: Adapters(a, b[:2]), lambda: Adapters(a, b.float()),
                lambda: Adapters(a[:, :4].contiguous(), b[:, :, :4].contiguous()), lambda: Adapters(a.cpu(), b.cpu()),
                lambda: Adapters(a, b.transpose(1, 2)), lambda: Adapters(a[:, :, :40].contiguous(), b),
                lambda: Adapters(a, b, scales.double()), lambda: Adapters(a, b, scales[:2]),
                lambda: Adapters(a.double(), b.double()), lambda: ok.add(y, xs[:, :32], ids),
                lambda: ok.add(y, xs, ids[:5]), lambda: ok.add(y, xs, ids.long()), lambda: ok.add(y.half(), xs, ids),
                lambda: ok.add(y[:5], xs, ids), lambda: ok.add(y, xs.double(), ids), lambda: ok.add(y, xs.cpu(), ids),
                lambda: ok.add(y.t().contiguous().t(), xs, ids), lambda: ok.add(y, xs, ids, out=y[:, :20]),
                lambda: Adapters.add_shared([y, y], xs, [ok], ids), lambda: Adapters.add_shared([], xs, [], ids),
                lambda: Adapters.add_shared([y, y], xs, [ok, other], ids),
                lambda: Adapters.add_shared([y] * 5, xs, [ok] * 5, ids),
                lambda: Adapters.add_shared([y, y], xs, [ok, ok], ids),
                lambda: Adapters.add_shared([y, other_y], xs, [ok, ok], ids, outs=[other_y, y]),
                lambda: Adapters(a, torch.zeros(3, 64, 8, device=DEV, dtype=a.dtype)).add(xs, xs, ids),
                lambda: Adapters.add_shared([y, other_y], xs, [ok, ok], ids, outs=[torch.empty_like(y), y])):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("rows,rank", [(3, 16), (20, 64), (1090, 64)])
def test_rows_far_apart(rows, rank):
    # x, y and out reach past 2^31 values (and 2^32 bytes)
    from swarmllm_amd import Adapters

    xs, a, b, scales, ids, y = make(5, rows, 1056, 72, rank, 3, "bf16")
    want, bound = ref.adapters(y, xs, ids, a, b, scales)
    step = (2 ** 31 // (rows - 1) + 64) // 8 * 8
    far_x = torch.empty(step * (rows - 1) + 1056, dtype=torch.bfloat16, device=DEV).as_strided((rows, 1056), (step, 1))
    far_y = torch.empty(step * (rows - 1) + 72, device=DEV).as_strided((rows, 72), (step, 1))
    far_x.copy_(xs)
    far_y.copy_(y)
    ad = Adapters(a, b, scales)
    close(ad.add(far_y, far_x, ids, out=torch.empty_like(y)), want, bound)
    assert torch.equal(ad.add(far_y, far_x, ids), ad.add(y, xs, ids))


def test_adapters_past_2_31_values():
    from swarmllm_amd import Adapters

    g = torch.Generator(device=DEV).manual_seed(8)
    slots, rank, k, n = 4096, 128, 4128, 2
    a = torch.empty(slots, rank, k, dtype=torch.bfloat16, device=DEV)
    b = torch.empty(slots, n, rank, dtype=torch.bfloat16, device=DEV)
    used = torch.tensor([0, 1, 4094, 4095], device=DEV)
    for i in used.tolist():
        a[i] = (torch.randn(rank, k, generator=g, device=DEV) / 64).bfloat16()
        b[i] = torch.randn(n, rank, generator=g, device=DEV).bfloat16()
    for rows in (2, 70, 4100):
        x = torch.randn(rows, k, generator=g, device=DEV)
        ids = used[torch.randint(4, (rows,), generator=g, device=DEV)].to(torch.int32)
        y = torch.randn(rows, n, generator=g, device=DEV)
        want, bound = ref.adapters(y, x, ids, a, b, None)
        close(Adapters(a, b).add(y, x, ids), want, bound)


def test_two_calls_at_once():
    from swarmllm_amd import Adapters

    sets = []
    for rows, k, rank in ((30, 2048, 64), (400, 8192, 64), (8, 4096, 16)):
        xs, a, b, scales, ids, y = make(rows, rows, k, 600, rank, 6)
        sets.append((Adapters(a, b, scales), xs, ids, y))
    want = [ad.add(y.clone(), xs, ids) for ad, xs, ids, y in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[] for _ in sets]
    torch.cuda.synchronize()
    for turn in range(5):
        for s, (ad, xs, ids, y), out in zip(streams, sets, outs):
            with torch.cuda.stream(s):
                out.append(ad.add(y.clone(), xs, ids))
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert all(torch.equal(o, w) for o in out)
