"""Adapters.add where single products show: their large parts cancel, so what a product leaves out is not hidden by
the sums' roundings. Rows one by one and in tiles of the matrix cores."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BITS = {"f32": 23, "f16": 10, "bf16": 7}
TYPES = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f32"), ("bf16", "f32"), ("f16", "f16")]


def left_out(one, other):
    """What a product may leave out of itself, by the types of its values."""
    if "bf16" in (one, other) or "f32" not in (one, other):
        return 0.0
    return 2.0 ** -23 if one == other else 2.0 ** -24


def just_past_one(g, shape, t):
    """Values 1 + r 2^-bits of type t, under 1 + 2^-7 (of bf16: 1 or 1 + 2^-7); some with every bit set."""
    bits = BITS[t]
    most = max(2, 1 << (bits - 7))
    r = torch.randint(most, shape, generator=g, device=DEV)
    r.view(-1)[::3] = most - 1
    return (1.0 + r.double() * 2.0 ** -bits).to(T[t])


@pytest.mark.parametrize("rows", [5, 1040])
@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("side", ["a", "b"])
def test_products_past_what_cancels(side, x, w, rows):
    # (1 + e)(1 + f) - 1 as two terms of one sum: in the matrix cores' instructions the two stand together, and
    # everything else that is added is at most 2^-5, so each of the 12 additions at most (six products of pieces,
    # three of the other side's ones, parts, the projection's 0) is off by half a step of that, 2^-29
    from swarmllm_amd import Adapters

    g = torch.Generator(device=DEV).manual_seed(rows + len(x) + 7 * len(w))
    n, rank, k, slots = 8, 8, 32, 2
    xs = torch.zeros(rows, k, dtype=T[x], device=DEV)
    xs[:, 3] = just_past_one(g, (rows,), x)
    xs[:, 17] = -1.0
    a = torch.zeros(slots, rank, k, dtype=T[w], device=DEV)
    b = torch.zeros(slots, n, rank, dtype=T[w], device=DEV)
    if side == "a":
        a[:, :, 3], a[:, :, 17] = just_past_one(g, (slots, rank), w), 1.0
        b[:] = torch.eye(8, device=DEV)
        factor = a[:, :, 3]
    else:
        a[:, 0, 3] = a[:, 5, 17] = 1.0
        b[:, :, 0], b[:, :, 5] = just_past_one(g, (slots, n), w), 1.0
        factor = b[:, :, 0]
    ids = torch.randint(slots, (rows,), generator=g, device=DEV).to(torch.int32)
    got = Adapters(a, b).add(torch.zeros(rows, n, device=DEV), xs, ids)
    product = xs[:, 3:4].double() * factor[ids.long()].double()
    off = (got.double() - (product - 1.0)).abs()
    if rows == 5:
        # one after another in fused additions: nothing is left out, and the sum is the product alone (1 to 1 + 2^-6)
        # before the other term comes, rounded by half a step of that, 2^-24
        out = 2.0 ** -24
    else:
        out = left_out(x if side == "a" else "f32", w)  # b's factors are f32 sums
    assert (off <= out * product + 12 * 2.0 ** -29).all(), float((off / product).max() * 2 ** 24)


@pytest.mark.parametrize("rows", [5, 1040])
@pytest.mark.parametrize("w", ["f32", "bf16"])
def test_values_next_to_the_largest(rows, w):
    # f32 values past the largest bf16 one, on either side of the product with b, come out finite
    from swarmllm_amd import Adapters

    g = torch.Generator(device=DEV).manual_seed(rows)
    n, rank, k = 16, 8, 32
    top = torch.finfo(torch.float32).max
    xs = torch.zeros(rows, k, device=DEV)
    xs[:, 9] = top * (1.0 - torch.rand(rows, generator=g, device=DEV) * 2.0 ** -7)
    xs[::2, 9] = top
    xs[::5] *= -1.0
    ids = torch.zeros(rows, dtype=torch.int32, device=DEV)
    for a_size, b_size in ((1.0, 2.0 ** -70), (2.0 ** -70, 1.0)):
        a = torch.zeros(1, rank, k, dtype=T[w], device=DEV)
        b = torch.zeros(1, n, rank, dtype=T[w], device=DEV)
        a[0, 4, 9], b[0, :, 4] = a_size, b_size
        got = Adapters(a, b).add(torch.zeros(rows, n, device=DEV), xs, ids)
        # powers of two: the value itself, from pieces that add up to it
        assert torch.equal(got.double(), (xs[:, 9:10].double() * 2.0 ** -70).expand(rows, n))
