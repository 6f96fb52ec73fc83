"""What a sequence's rows may take from the other sequences of its call: from
their values and pages nothing; from their lengths, at most the last bits of a
row, and those only where more than 256 query rows a kv head are planned."""
import pytest
import torch

from layer_reference import attend64
from test_attend_gpu import F16, F32, batch, check

pytestmark = pytest.mark.gpu

# (new tokens, cached) of three sequences, other lengths of the first and last, heads, kv heads, the one looked at alike
CALLS = {
    "few": ([1, 3, 2], [300, 500, 100], [3, 3, 0], [7, 500, 500], 8, 2),
    "few in parts": ([1, 3, 2], [9000, 8000, 100], [3, 3, 0], [7, 8000, 9000], 8, 2),
    "chunk": ([20, 40, 9], [300, 500, 100], [1, 40, 40], [500, 500, 45], 8, 2),
    "chunk in parts": ([60, 40, 9], [5000, 4100, 100], [1, 40, 0], [500, 4100, 0], 8, 2),
    "blocks of 256 rows in parts": ([300, 290, 9], [5000, 4100, 100], [1, 290, 200], [500, 4100, 4000], 4, 4),
}
SHARES = ([1100, 700, 600], [2600, 2100, 700], [30, 700, 1], [90, 2100, 2500], 40, 40)


def both(new, kvl, other_new, other_kvl, heads, kv_heads, seed, dtype=F32):
    """The middle sequence's rows of a call, of one with other values beside it, and of one with other lengths."""
    kv, q, starts, lens, tables, _ = batch(new, kvl, heads, kv_heads, 64, 32, dtype, seed=seed, spare=300)
    max_q, max_kv = max(new), max(kvl)

    def middle(n, k, x, table):
        s = torch.tensor([0, n[0], n[0] + n[1], sum(n)], dtype=torch.int32, device="cuda")
        out = kv.attend(x, s, torch.tensor(k, dtype=torch.int32, device="cuda"), table, max_q=max_q, max_kv=max_kv)
        return out[n[0]: n[0] + n[1]]

    mine = q[new[0]: new[0] + new[1]]
    first = middle(new, kvl, q, tables)
    assert torch.equal(middle(new, kvl, q, tables), first)
    x = torch.randn_like(q)
    x[new[0]: new[0] + new[1]] = mine
    moved = tables.clone()
    moved[0], moved[2] = tables[2], tables[0]
    values = middle(new, kvl, x, moved)
    x = torch.randn(sum(other_new), *q.shape[1:], device="cuda").to(dtype)
    x[other_new[0]: other_new[0] + other_new[1]] = mine
    lengths = middle(other_new, other_kvl, x, tables)
    want, tol = attend64(kv, mine, torch.tensor([0, new[1]]), torch.tensor(kvl[1:2]), tables[1:2], 0.125)
    return first, values, lengths, want, tol


@pytest.mark.parametrize("call", CALLS)
def test_rows_are_the_same_bits_beside_other_values_and_lengths(call):
    first, values, lengths, want, tol = both(*CALLS[call], seed=len(call))
    check(first, want, tol)
    assert torch.equal(values, first) and torch.equal(lengths, first)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_chunks_in_equal_shares(dtype):
    """The same bits beside other values; beside other lengths within the roundings, wherever the shares end."""
    first, values, lengths, want, tol = both(*SHARES, seed=1, dtype=dtype)
    assert torch.equal(values, first)
    check(first, want, tol)
    check(lengths, want, tol)
