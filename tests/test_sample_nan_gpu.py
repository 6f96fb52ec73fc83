"""A NaN among a row's settings turns that setting off, whatever others are on and however many values they leave:
the same token and chance as of a row without it."""
import math

import pytest
import torch

import batch_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("vocab", [300, 5000, 128256])
@pytest.mark.parametrize("name,values", [("top_k", [1, 5, 40, 64, 65, 200, 700, 1500, 3000]),
                                         ("min_p", [1.0, 0.3, 0.05, 1e-2, 1e-3, 1e-4, 1e-6]), ("temperature", [0.0, 0.5, 1.0, 3.0])])
def test_nan_top_p_beside_another_setting(name, values, vocab):
    import swarmllm_amd as sa

    g = torch.Generator(device=DEV).manual_seed(vocab)
    rows = 8 * len(values)
    x = 2.2 * torch.randn(rows, vocab, generator=g, device=DEV)
    u = torch.linspace(0.02, 0.98, rows, device=DEV)
    beside = torch.tensor(values, dtype=torch.int32 if name == "top_k" else torch.float32, device=DEV).repeat(8)
    nan = torch.full((rows,), math.nan, device=DEV)
    want = sa.sample(x, u, **{name: beside})
    got = sa.sample(x, u, top_p=nan, **{name: beside})
    assert torch.equal(got.ids, want.ids) and torch.equal(got.probs, want.probs)
    for r in range(rows):
        w = ref.kept(x[r], **{name: beside[r].item(), "top_p": math.nan})
        want_id, chance = ref.token(w, u[r].item())
        assert got.ids[r].item() == want_id, (r, beside[r].item())
        # one rounding to f32, and 64-bit sums
        assert abs(got.probs[r].item() - chance) <= 2.0 ** -23 * chance, (r, beside[r].item())


def test_nan_min_p_and_temperature_beside_others():
    import swarmllm_amd as sa

    g = torch.Generator(device=DEV).manual_seed(1)
    x, u = 2.2 * torch.randn(12, 40000, generator=g, device=DEV), torch.linspace(0.02, 0.98, 12, device=DEV)
    nan, p = torch.full((12,), math.nan, device=DEV), torch.full((12,), 0.9, device=DEV)
    k = torch.tensor([0, 5, 40, 200, 700, 3000] * 2, dtype=torch.int32, device=DEV)
    for a, b in ((sa.sample(x, u, top_k=k, top_p=p, min_p=nan), sa.sample(x, u, top_k=k, top_p=p)),
                 (sa.sample(x, u, temperature=nan, top_k=k, top_p=p), sa.sample(x, u, temperature=0 * p))):
        assert torch.equal(a.ids, b.ids) and torch.equal(a.probs, b.probs)
