"""sample where thousands of values lie at the border of top_p and each weighs next to nothing beside the largest
one: the run has to end where the sums in 64 bits say. With u = 1 and values that fall with their index the token is
the run's last value itself."""
import pytest
import torch

import batch_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("vocab,low", [(524288, -21.5), (128256, -23.6)])
@pytest.mark.parametrize("equal", [False, True])
@pytest.mark.parametrize("part", [0.3, 0.5, 0.8])
def test_the_run_s_last_value(vocab, low, equal, part):
    import swarmllm_amd as sa

    x = torch.full((vocab,), low, device=DEV)
    if not equal:
        x += torch.linspace(0.5, -0.5, vocab, device=DEV)
    x[0] = 0.0
    rest = float(x.double().exp().sum()) - 1.0
    rows = 4
    p = torch.tensor([(1.0 + (part + 0.01 * r) * rest) / (1.0 + rest) for r in range(rows)], device=DEV)
    assert (p < 1.0).all() and p.unique().numel() == rows
    u = torch.ones(rows, device=DEV)
    for top_k in (0, vocab - 1, vocab - vocab // 16):
        k = torch.full((rows,), top_k, dtype=torch.int32, device=DEV)
        got = sa.sample(x.expand(rows, vocab).contiguous(), u, None, k, p).ids.tolist()
        for r in range(rows):
            w = ref.kept(x, 1.0, top_k, p[r].item())
            want = int(torch.nonzero(w > 0)[-1])
            # two sums of at most 2^19 terms, each addition off by half a step of 64 bits of at most the
            # total: 2^-33 of it together, at 128256 terms 2^-35, and a value at the border weighs more: 2^-32 and 2^-35
            assert abs(got[r] - want) <= 1, (top_k, r, got[r], want)
