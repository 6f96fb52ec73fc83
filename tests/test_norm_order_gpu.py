"""The sum of squares of rms_norm_act runs in one order, whatever launch a
row's batch gets: rows whose mean square stands so near the border between two
f32 values of rs that the order of a 64-bit sum decides."""
import numpy as np
import pytest
import torch

from swarmllm_amd import rms_norm_act

pytestmark = pytest.mark.gpu


def sum_of_squares(row, waves):
    """In 64 bits, as `waves` waves do that take blocks of 256 values in turn: a lane's 4 of each block, the lanes
    by exchange (32, 16, .. 1), the waves from the first on. (A square of an f32 is exact in 64 bits.)"""
    blocks = np.zeros((-(-len(row) // (256 * waves)) * waves, 64, 4))
    blocks.reshape(-1)[: len(row)] = row.astype(np.float64)
    s = np.zeros((waves, 64))
    for b in range(len(blocks)):
        for i in range(4):
            s[b % waves] += blocks[b, :, i] ** 2
    for m in (32, 16, 8, 4, 2, 1):
        s = s + s[:, np.arange(64) ^ m]
    total = 0.0
    for w in range(waves):
        total += s[w, 0]
    return total


def rs(ss, k):
    return np.float32(1.0 / np.sqrt(ss / k))


def row_at_a_border(k, seed):
    """A row whose rs differs between sums by 4 and by 16 waves: one large value, many whose squares are under half
    a step of its square's 64 bits (lost one by one, kept when added up first), and two that bring the sum to the border."""
    rng = np.random.default_rng(seed)
    for _ in range(40):
        big = np.float32(rng.uniform(40.0, 60.0))
        row = np.full(k, np.float32(float(big) * 2.0**-27), dtype=np.float32)
        row[[0, 8, 12]] = big, 0.0, 0.0
        low = np.nextafter(rs(sum_of_squares(row, 16), k), np.float32(0))
        border = k / ((float(low) + float(np.nextafter(low, np.float32(0)))) / 2) ** 2
        for step in range(-24, 8):
            left = border * (1 + step * 2.0**-53) - sum_of_squares(row, 16)
            near = row.copy()
            near[8] = np.float32(np.sqrt(left) * (1 - 2.0**-24))
            if float(near[8]) ** 2 > left:
                near[8] = np.nextafter(near[8], np.float32(0))
            near[12] = np.float32(np.sqrt(max(left - float(near[8]) ** 2, 0.0)))
            if rs(sum_of_squares(near, 4), k) != rs(sum_of_squares(near, 16), k):
                return near
    raise AssertionError("no such row found")


@pytest.mark.parametrize("k", [1280, 4096, 8192])
def test_the_order_of_the_sum_does_not_follow_from_the_batch(k):
    row = torch.from_numpy(row_at_a_border(k, k)).cuda()
    w = torch.ones(k, device="cuda")
    one = rms_norm_act(row[None], w, 0.0, y_dtype=torch.float32)
    many = rms_norm_act(row.expand(600, k).contiguous(), w, 0.0, y_dtype=torch.float32)
    assert (many.y == one.y).all()
    for a, b in zip(one.act.planes(), many.act.planes()):
        assert (a[0] == b).all()


def test_more_rows_than_a_launch_has_threads_in_one_direction():
    """2^26 rows of a wave each, and some."""
    rows = 2**26 + 5
    x = torch.arange(rows, device="cuda", dtype=torch.int32).remainder_(251).add_(1).float()[:, None].repeat(1, 4)
    x[:, 1] = 0.5
    out = rms_norm_act(x, torch.ones(4, device="cuda"), 0.0, dtype=None, y_dtype=torch.float32)
    for part in (slice(0, 2000), slice(2**25 - 1000, 2**25 + 1000), slice(rows - 2000, rows)):
        h = x[part].double()
        want = h / h.square().mean(1, keepdim=True).sqrt()
        assert ((out.y[part].double() - want).abs() <= 3.001 * 2.0**-24 * want).all()
    # and no row is another's
    assert torch.equal(out.y[:251].repeat(3, 1), out.y[251 * 2**17: 251 * (2**17 + 3)])
