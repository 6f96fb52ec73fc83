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
