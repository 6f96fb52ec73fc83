"""Adapters.add beside memory that other arrays share: refused where a byte is in common (and nothing is written),
right where rows only lie between each other's."""
import pytest
import torch

import batch_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rows", [3, 40, 1100])
def test_shared_memory(rows):
    from swarmllm_amd import Adapters

    g = torch.Generator(device=DEV).manual_seed(rows)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    k, n = 64, 64
    ads = [Adapters(rand(3, 8, k).bfloat16(), rand(3, n, 8).bfloat16(), rand(3)) for _ in range(2)]
    ids = torch.randint(-1, 3, (rows,), generator=g, device=DEV).to(torch.int32)
    flat = rand(3 * rows * n + 64)
    before = flat.clone()
    y, near = flat[:rows * n].view(rows, n), flat[8:8 + rows * n].view(rows, n)
    late = flat[rows * n:2 * rows * n].view(rows, n)
    x = rand(rows, k)
    for bad in (lambda: ads[0].add(y, x, ids, out=near), lambda: ads[0].add(near, x, ids, out=y),
                lambda: ads[0].add(late, y, ids, out=near), lambda: ads[0].add(y, y, ids),
                lambda: ads[0].add(late, near, ids, out=y),
                lambda: Adapters.add_shared([y, near], x, ads, ids),
                lambda: Adapters.add_shared([y, late], x, ads, ids, outs=[late, flat[2 * rows * n:3 * rows * n].view(rows, n)]),
                lambda: Adapters.add_shared([y, late], x, ads, ids, outs=[near, late])):
        with pytest.raises(ValueError):
            bad()
    assert torch.equal(flat, before)
    # columns of one wide array: x, two projections' y in place, and a strip that stays
    wide = rand(rows, k + 2 * n + 20)
    left = wide.clone()
    xs, ys = wide[:, 4:4 + k], [wide[:, k + 8:k + 8 + n], wide[:, k + n + 12:k + 2 * n + 12]]
    want = [ref.adapters(v.clone(), xs.clone(), ids, ad.a, ad.b, ad.scales) for v, ad in zip(ys, ads)]
    Adapters.add_shared(ys, xs, ads, ids)
    for v, (w, bound) in zip(ys, want):
        assert ((v.double() - w).abs() <= bound).all()
    for a, b in ((0, k + 8), (k + 8 + n, k + n + 12), (k + 2 * n + 12, k + 2 * n + 20)):
        assert torch.equal(wide[:, a:b], left[:, a:b])
