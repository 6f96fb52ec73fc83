"""Elementwise steps of more values than one direction of a launch has threads."""
import pytest
import torch

from swarmllm_amd import glu

pytestmark = pytest.mark.gpu


def test_more_gated_values_than_a_launch_has_threads_in_one_direction():
    """2^32 values and some: the gated activation of a long prompt's batch, as forward_glu's second step takes it."""
    n = 2**32 + 1000
    gate, up = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    some = [slice(0, 3000), slice(2**31 - 500, 2**31 + 500), slice(n - 3000, n)]
    for s in some:
        gate[s], up[s] = (torch.randn(s.stop - s.start, device="cuda") for _ in range(2))
    out = glu(gate, up)
    for s in some:
        assert torch.equal(out[s], glu(gate[s].clone(), up[s].clone())) and out[s].abs().sum() > 0
    assert not out[2**31 + 500: 2**31 + 10**6].any()
