"""Attention whose scores lie far from zero, against 64 bits.

Queries and cached keys are small whole numbers (times a power of two), so every
f16 operand and every f32 score is exact, and what is left to allow for is the
same at any scale: a weight and a value round to f16 (2^-11 each), a weight
below 2^-14 by 2^-25, f32 sums over n positions by n / 64 + 64 steps of 2^-24,
and the maxima that sums are relative to, times the scale, by 2^-17 of an
exponent of 2 each side of a join, in the sums above and below the line: 4 ln 2
2^-17 < 2^-15. The scales are f32 numbers."""
import pytest
import torch

from layer_reference import attend64, rounding
from swarmllm_amd import KvCache
from test_attend_gpu import BF16, F16, F32, batch

pytestmark = pytest.mark.gpu


def whole_keys(kv, g, power=1.0):
    kv.planes[0].copy_(torch.randint(-127, 128, kv.planes[0].shape, generator=g, device="cuda"))
    kv.planes[1].fill_(power)


def check_exact_scores(kv, q, starts, lens, tables, scale, sinks=None, **how):
    got = kv.attend(q, starts, lens, tables, scale=scale, sinks=sinks, **how)
    want, _ = attend64(kv, q, starts, lens, tables, scale, 0, sinks)
    codes = kv.planes[2].clone()
    kv.planes[2].abs_()
    size, _ = attend64(kv, q, starts, lens, tables, scale, 0, sinks)
    top = float((kv.planes[2].float().amax() * kv.planes[3].float().amax()))
    kv.planes[2].copy_(codes)
    n, u = int(lens.max()), 2.0**-11
    tol = (2 * u * (1 + u) + (n / 64 + 64) * 2.0**-24 + 2.0**-15) * size + 2.0**-25 * n * top
    err = (got.double() - want).abs()
    ok = err <= tol + rounding(got.dtype) * (want.abs() + tol) + 2.0**-25
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} off, got {got[~ok][:4].tolist()} want {want[~ok][:4].tolist()}"


SCALES = [0.375, 8.0, -8.0, 2.0**24, -(2.0**40), 2.0**64, 2.0**99, -(2.0**99)]


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("new,kvl,heads,kv_heads,hd,page,dtype", [
    ([1, 2, 3], [700, 500, 64], 4, 2, 64, 64, F16),       # few rows, whole
    ([1], [9001], 8, 1, 128, 64, F32),                    # few rows, in parts
    ([40, 1], [600, 300], 4, 2, 128, 16, BF16),           # a chunk
    ([40], [5000], 8, 1, 96, 32, F16),                    # a chunk in parts
    ([300], [2300], 8, 1, 64, 64, F16),                   # blocks of 256 rows
    ([33, 7], [400, 90], 4, 2, 256, 128, F16),
])
def test_whole_scores_of_any_scale(scale, new, kvl, heads, kv_heads, hd, page, dtype):
    for sinks in (False, True):
        kv, q, starts, lens, tables, sk = batch(new, kvl, heads, kv_heads, hd, page, dtype, seed=hd, sinks=sinks)
        g = torch.Generator(device="cuda")
        g.manual_seed(int(sum(kvl)))
        whole_keys(kv, g)
        q = torch.randint(-3, 4, q.shape, generator=g, device="cuda").to(dtype)
        check_exact_scores(kv, q, starts, lens, tables, scale, sk, max_q=max(new))


@pytest.mark.parametrize("scale", [8.0, 2.0**99, -(2.0**40)])
def test_whole_scores_of_any_scale_in_shares(scale):
    new, kvl = [1100, 1, 700, 300, 430], [2300, 2100, 700, 2600, 200]
    kv, q, starts, lens, tables, sk = batch(new, kvl, 20, 20, 64, 64, F16, seed=3, sinks=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    whole_keys(kv, g)
    q = torch.randint(-3, 4, q.shape, generator=g, device="cuda").to(F16)
    check_exact_scores(kv, q, starts, lens, tables, scale, sk, max_q=1100)


@pytest.mark.parametrize("new,n", [(1, 900), (1, 9000), (60, 900), (300, 2500)])
def test_queries_and_keys_in_the_thousands(new, n):
    """4000 times up to 4064 in each of 128 dims, the scale of that many (an f32 number): scores of 10^8."""
    kv, q, starts, lens, tables, _ = batch([new], [n], 4, 1, 128, 64, F16, seed=n)
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    kv.planes[0].copy_(torch.randint(-127, 128, kv.planes[0].shape[:3], generator=g, device="cuda")[..., None]
                       .expand(kv.planes[0].shape))
    kv.planes[1].fill_(32.0)
    q.fill_(4000.0)
    q[:, 1::2] = -4000.0
    check_exact_scores(kv, q, starts, lens, tables, 0.0883883461356163, max_q=new)


@pytest.mark.parametrize("new,n", [(1, 90), (1, 9000), (40, 600), (40, 5000)])
def test_sinks_past_the_largest_number(new, n):
    """A sink that is infinite, or is so in the exponent's base, takes all of a row's weight; one below every number none."""
    kv, q, starts, lens, tables, _ = batch([new], [n], 4, 2, 64, 64, F32, seed=n)
    none = kv.attend(q, starts, lens, tables, max_q=new)
    inf = float("inf")
    got = kv.attend(q, starts, lens, tables, max_q=new, sinks=torch.tensor([inf, 3e38, -inf, -3e38], device="cuda"))
    assert (got[:, :2] == 0).all() and torch.equal(got[:, 2:], none[:, 2:])
    far = kv.attend(q, starts, lens, tables, max_q=new, scale=2.0**99, sinks=torch.full((4,), inf, device="cuda"))
    assert (far == 0).all()


@pytest.mark.parametrize("new", [1, 33])
def test_many_small_weights_beside_a_large_one(new):
    """2^20 positions of a weight of 2^-25.5 behind one of 1: together 2 % of the row, and each under half the smallest
    f16. 64 sequences of 8 kv heads on the same pages, so that none is cut in parts that would each find a maximum of
    its own. The weak weights are exact to 2^-32 (half the smallest f16, the weights lifted by 2^7)."""
    n, seqs, page = 2**20, 64, 256
    kv = KvCache.alloc(n // page, 8, 64, page)
    kv.planes[1].fill_(1.0)
    kv.planes[3].fill_(2.0**-7)
    kv.planes[0][..., 0] = -51
    kv.planes[0][0, :, 0, 0] = 0
    v = torch.randint(-127, 128, (8, 64), device="cuda", dtype=torch.int8)
    first = torch.randint(-127, 128, (8, 64), device="cuda", dtype=torch.int8)
    kv.planes[2][:] = v[None, :, :, None]
    kv.planes[2][0, :, :, 0] = first
    q = torch.zeros(seqs * new, 8, 64, device="cuda")
    q[..., 0] = 1.0
    scale = 0.34657359  # ln 2 / 2 (as an f32 number): 51 of it are 25.5 powers of two
    scale32 = torch.tensor(scale, dtype=torch.float32).double()
    starts = torch.arange(seqs + 1, device="cuda", dtype=torch.int32) * new
    lens = torch.full((seqs,), n, device="cuda", dtype=torch.int32)
    tables = torch.arange(n // page, device="cuda", dtype=torch.int32).expand(seqs, -1).contiguous()
    got = kv.attend(q, starts, lens, tables, max_q=new, scale=scale)
    w = torch.exp(-51.0 * scale32.cuda())
    weak = w * (n - new + torch.arange(new, device="cuda").double()).repeat(seqs)[:, None, None]
    want = (first.double() + weak * v.double()) * 2.0**-7 / (1 + weak)
    size = (first.double().abs() + weak * v.double().abs()) * 2.0**-7 / (1 + weak)
    # 2^-11 a value and a weight, 2^-15 the exponents and joins, a weak weight 2^-32. The matrix instructions add 8
    # positions' products to a sum at a time and round it to nearest, by at most 2^-24 of itself, each time (16 products of
    # 1/16, 3/16 and 5/16 of a step of the sum add 0, 4 and 4 steps: two eights of 1/2, 3/2 and 5/2, to even). That is n / 8
    # times for a chunk's row and n / 32 times in each of the four waves of few rows, and up to 64 more in joins; here all to
    # one side, for each addition is the same 8 weights of 2^-18.5 (1.4 |v| / |first| of the sum's steps). 0.8 % of a row, 0.2
    adds = (n / 8 if new > 32 else n / 32) + 64
    tol = (2 * 2.0**-11 * (1 + 2.0**-11) + 2.0**-15 + 2.0**-24 * adds) * size + 2.0**-32 * n
    assert ((got.double() - want).abs() <= tol + rounding(F32) * want.abs()).all(), float(((got.double() - want).abs() - tol).max())
