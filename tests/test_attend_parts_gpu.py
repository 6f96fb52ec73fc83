"""Attention whose blocks are left over behind the last whole round of the CUs
and cut into parts: some heads' blocks of a row of them, whole rows and some of
the next, none. Against 64 bits (layer_reference.attend64)."""
import pytest
import torch

from layer_reference import attend64
from test_attend_gpu import BF16, F16, batch, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,new,n,heads,kv_heads,hd,page,dtype", [
    (65, 5, 2100, 64, 8, 64, 64, F16),      # 520 blocks of 128 rows: 8 left
    (7, 200, 4000, 40, 40, 64, 32, BF16),   # 560: 48 left, of the second row
    (10, 850, 1100, 10, 10, 64, 64, F16),   # 700: 188 left, the first row's 100 and 88 of the second's
    (9, 300, 2200, 12, 12, 256, 64, F16),   # 324 with 256 CUs' worth a round: 68 left of the first row's 108
    (3, 1100, 2400, 20, 20, 128, 64, F16),  # blocks of 256 rows
])
@pytest.mark.parametrize("window,sinks", [(0, True), (500, False)])
def test_blocks_left_behind_the_last_round(seqs, new, n, heads, kv_heads, hd, page, dtype, window, sinks):
    lens = [n - 37 * b % 400 for b in range(seqs)]
    news = [max(1, new - 3 * (b % 5) * (b % 2)) for b in range(seqs)]
    kv, q, starts, kv_lens, tables, sk = batch(news, lens, heads, kv_heads, hd, page, dtype, seed=seqs, sinks=sinks)
    got = kv.attend(q, starts, kv_lens, tables, max_q=new, window=window, sinks=sk)
    check(got, *attend64(kv, q, starts, kv_lens, tables, hd ** -0.5, window, sk))
    again = kv.attend(q, starts, kv_lens, tables, max_q=new, window=window, sinks=sk)
    assert torch.equal(got, again)
