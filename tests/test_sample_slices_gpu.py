"""sample's rows in slices: a row's workgroups hand their results to the last of them, so a row has to come out the
same whether one workgroup has it (many rows) or eight (few), call after call."""
import pytest
import torch

import batch_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("vocab", [32000, 128256])
def test_rows_in_any_number_of_slices(vocab):
    import swarmllm_amd as sa

    rows = 600
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = 2.2 * torch.randn(rows, vocab, generator=g, device=DEV)
    u = torch.rand(rows, generator=g, device=DEV)
    t = 0.7 + torch.rand(rows, generator=g, device=DEV)
    at = torch.arange(rows, device=DEV)
    p = torch.tensor([0.9, 0.5, 0.999, 0.95], device=DEV)[at % 4]
    k = torch.tensor([0, 0, 0, 0, 700, 450, 3000], dtype=torch.int32, device=DEV)[at % 7].contiguous()
    m = torch.tensor([0.0, 1e-5, 0.0], device=DEV)[at % 3]
    one = torch.ones_like(p)
    for settings in ((t, None, p, None), (t, k, torch.where(k > 0, one, p), None), (t, None, None, m + 1e-6), (t, k, p, m)):
        whole = sa.sample(x, u, *settings)
        for r in (0, 5, 11, 301, 599):
            f = [v[r].item() if v is not None else off for v, off in zip(settings, (1.0, 0, 1.0, 0.0))]
            want, chance = ref.token(ref.kept(x[r], *f), u[r].item())
            assert whole.ids[r].item() == want, (r, f)
            assert abs(whole.probs[r].item() - chance) <= 2.0 ** -23 * chance
        for count in (1, 3, 16, 33, 64, 128, 200):
            for first in (0, 300, 600 - count):
                s = slice(first, first + count)
                got = sa.sample(x[s], u[s], *(v[s] if v is not None else None for v in settings))
                assert torch.equal(got.ids, whole.ids[s]), (count, first)
                # one rounding to f32 each
                assert ((got.probs - whole.probs[s]).abs() <= 2.0 ** -23 * whole.probs[s]).all(), (count, first)
