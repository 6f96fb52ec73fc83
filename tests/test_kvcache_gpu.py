"""The paged Q8_0 cache: writes against the CPU oracle's Q8_0 wire blocks bit
for bit (codes and scales, every other slot of the cache untouched), reads
against code * scale rounded once."""
import numpy as np
import pytest
import torch

from layer_reference import wire_blocks
from swarmllm_amd import KvCache

pytestmark = pytest.mark.gpu


def noise(kv, seed):
    """Fills the planes, so that a write beside its slots shows."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    for t in kv.planes:
        if t.dtype == torch.int8:
            t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda", dtype=torch.int8))
        else:
            t.copy_(torch.rand(t.shape, generator=g, device="cuda"))


TOP = 65468.5  # 127 * 515.5: the f16 after 515.5 is 516, and 127 * 516 = 65532 rounds to an infinite f16


def expect_write(kv, k, v, slots):
    """The planes after the write, from the oracle (finite values cut at TOP first)."""
    kc, ks, vc, vs = (t.cpu().numpy().copy() for t in kv.planes)
    for x, codes, scales, tr in ((k, kc, ks, False), (v, vc, vs, True)):
        x = x.float()
        q, d = wire_blocks(torch.where(x.isfinite(), x.clamp(-TOP, TOP), x).cpu().numpy())
        for t, s in enumerate(slots.tolist()):
            if not 0 <= s < kv.pages * kv.page:
                continue
            p, o = divmod(s, kv.page)
            if tr:
                codes[p, :, :, o], scales[p, :, :, o] = q[t], d[t]
            else:
                codes[p, :, o], scales[p, :, o] = q[t], d[t]
    return kc, ks, vc, vs


def check(kv, want):
    for t, w in zip(kv.planes, want):
        assert np.array_equal(t.cpu().numpy().view(np.uint8), w.view(np.uint8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,heads,hd,page", [(1, 8, 128, 64), (1, 1, 64, 16), (7, 2, 96, 32), (8, 8, 128, 64),
                                                  (33, 3, 256, 16), (130, 2, 64, 128), (300, 8, 128, 64),
                                                  (257, 1, 96, 256)])
def test_write_and_read(dtype, tokens, heads, hd, page):
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens + hd)
    pages = -(-tokens // page) + 2
    kv = KvCache.alloc(pages, heads, hd, page)
    for order in ("runs", "scattered"):
        noise(kv, tokens)
        if order == "runs":  # whole pages in any order, the last one in part
            table = torch.randperm(pages, generator=g, device="cuda")
            slots = kv.slots(table, 0, tokens)
        else:
            slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].contiguous()
        # slices of one fused row, as a product writes them
        rows = (torch.randn(tokens, 4 * heads * hd, generator=g, device="cuda") * 3).to(dtype)
        k = rows[:, heads * hd: 2 * heads * hd].unflatten(1, (heads, hd))
        v = rows[:, 3 * heads * hd:].unflatten(1, (heads, hd))
        want = expect_write(kv, k, v, slots)
        kv.write(k, v, slots)
        check(kv, want)
        kc, ks, vc, vs = kv.planes
        p, o = slots // page, slots % page
        k32 = (kc[p, :, o].float().unflatten(2, (-1, 32)) * ks[p, :, o].float()[..., None]).flatten(2)
        v32 = (vc[p, :, :, o].float().unflatten(2, (-1, 32)) * vs[p, :, :, o].float()[..., None]).flatten(2)
        for t in (torch.float32, torch.float16, torch.bfloat16):
            a, b = kv.read(slots, t)
            assert torch.equal(a, k32.to(t)) and torch.equal(b, v32.to(t))


@pytest.mark.parametrize("start", [0, 1, 5, 16, 61])
@pytest.mark.parametrize("tokens", [2, 16, 50, 64, 200])
def test_runs_that_begin_and_end_inside_a_page(start, tokens):
    """A chunk appended behind `start` tokens: pieces of pages at both ends."""
    g = torch.Generator(device="cuda")
    g.manual_seed(start * 100 + tokens)
    kv = KvCache.alloc(8, 2, 64, 64)
    noise(kv, 5)
    slots = kv.slots(torch.randperm(8, generator=g, device="cuda"), start, tokens)
    k, v = (torch.randn(tokens, 2, 64, generator=g, device="cuda") for _ in range(2))
    want = expect_write(kv, k, v, slots)
    kv.write(k, v, slots)
    check(kv, want)
    a, b = kv.read(slots, torch.float32)
    for i in (0, tokens - 1):
        x, y = kv.read(slots[i:i + 1], torch.float32)
        assert torch.equal(x[0], a[i]) and torch.equal(y[0], b[i])


def test_padding_slots_write_nothing_and_read_zeros():
    kv = KvCache.alloc(3, 2, 64, 16)
    noise(kv, 1)
    k, v = (torch.randn(20, 2, 64, device="cuda") for _ in range(2))
    slots = torch.tensor([-1, 47, 48, 0, -(2**40), 2**40, 5, 6, -1, 7] + list(range(16, 26)), device="cuda")
    want = expect_write(kv, k, v, slots)
    kv.write(k, v, slots)
    check(kv, want)
    a, b = kv.read(slots)
    out = (slots < 0) | (slots >= 48)
    assert (a[out] == 0).all() and (b[out] == 0).all() and a[~out].abs().sum() > 0
    # a slot may be read twice
    a, b = kv.read(torch.tensor([5, 5, 47, 5], device="cuda"))
    assert torch.equal(a[0], a[1]) and torch.equal(b[0], b[3])


def test_special_values():
    """Zeros, infinities, NaN, values past f16's range, subnormal scales."""
    kv = KvCache.alloc(2, 1, 64, 16)
    noise(kv, 2)
    x = torch.zeros(8, 1, 64, device="cuda")
    x[1, 0, 3], x[1, 0, 4], x[1, 0, 5] = float("inf"), float("-inf"), float("nan")
    x[1, 0, 6] = 2.0
    x[2] = float("nan")
    x[3] = 1e-30
    x[4] = 1e-7
    x[5, 0, :32] = 65504.0
    x[6, 0, 32:] = torch.linspace(-1, 1, 32, device="cuda")
    x[7] = 2.5
    slots = torch.arange(8, device="cuda")
    want = expect_write(kv, x, x, slots)
    kv.write(x, x, slots)
    check(kv, want)
    big = torch.full((1, 1, 64), 1e30, device="cuda")
    big[0, 0, 7] = -70000.0
    kv.write(big, big, slots[:1])
    a, b = kv.read(slots[:1], torch.float32)
    assert torch.equal(a.abs(), torch.full_like(a, TOP)) and a[0, 0, 7] == -TOP and torch.equal(a, b)
    assert torch.isfinite(kv.read(slots[:1], torch.float16)[0]).all()


@pytest.mark.parametrize("heads,hd,page", [(8, 128, 64)])
def test_slots_past_32_bit_offsets(heads, hd, page):
    pages = 2**32 // (page * heads * hd) + 3  # a codes plane of more than 4 GiB
    kv = KvCache.alloc(pages, heads, hd, page)
    slots = torch.tensor([0, 5, (2**31) // (heads * hd) + 1, pages * page - 1, pages * page - page], device="cuda")
    k, v = (torch.randn(5, heads, hd, device="cuda") for _ in range(2))
    kv.write(k, v, slots)
    a, b = kv.read(slots, torch.float32)
    for x, got in ((k, a), (v, b)):
        q, d = wire_blocks(x.cpu().numpy())
        want = (q.reshape(5, heads, -1, 32).astype(np.float32) * d.astype(np.float32)[..., None]).reshape(x.shape)
        assert np.array_equal(got.cpu().numpy(), want)
    assert int((kv.planes[0][torch.unique(slots // page)] != 0).sum()) == int((a != 0).sum())


def test_refusals():
    kv = KvCache.alloc(3, 2, 64, 16)
    k = torch.randn(4, 2, 64, device="cuda")
    s = torch.arange(4, device="cuda")
    for bad in (lambda: kv.write(k, k, s.int()), lambda: kv.write(k, k, s[:3]), lambda: kv.write(k, k.half(), s),
                lambda: kv.write(k[:, :1], k, s), lambda: kv.write(k.double(), k.double(), s),
                lambda: kv.write(k.cpu(), k.cpu(), s), lambda: kv.write(k.transpose(1, 2).contiguous().transpose(1, 2), k, s),
                lambda: kv.write(k, k, s[::2]), lambda: kv.read(s.cpu()), lambda: kv.read(s, torch.float64),
                lambda: kv.write(k[:, :, :32], k[:, :, :32], s), lambda: KvCache.alloc(3, 2, 80),
                lambda: KvCache.alloc(3, 2, 64, 24), lambda: KvCache.alloc(3, 2, 64, 512), lambda: KvCache.alloc(0, 2, 64),
                lambda: KvCache.alloc(3, 0, 64), lambda: KvCache(*(t.cpu() for t in kv.planes)),
                lambda: KvCache(kv.planes[0], kv.planes[1], kv.planes[0], kv.planes[3]),
                lambda: KvCache(kv.planes[0][:, :, :, ::2], *kv.planes[1:])):
        with pytest.raises(ValueError):
            bad()
    kv.write(k[:0], k[:0], s[:0])
    assert kv.read(s[:0])[0].shape == (0, 2, 64)
