"""Eviction at the largest numbers of slices."""

from __future__ import annotations

import pytest
import torch

from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("capacity", [1, 2])
def test_more_slices_than_one_grid_has_threads_for(capacity):
    """4194304 workgroups of 1024 threads are 2^32: more than one launch takes."""
    from dilution import kernels

    n, length, d = 4194304 + 5, 3, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(n, 1, length, d, generator=g, device="cuda").to(torch.bfloat16)
    v = torch.randn(n, 1, length, d, generator=g, device="cuda").to(torch.bfloat16)
    com = torch.rand(n, 1, length, generator=g, device="cuda")
    ko, vo, co, index = kernels.dilution_evict(k, v, com, length, 1, capacity=capacity)
    # the first of the largest: later keys only where they hold more
    best = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    most = com[..., 0].clone()
    for j in (1, 2):
        more = com[..., j] > most
        best[more], most[more] = j, com[..., j][more]
    assert torch.equal(index[..., 0], best)
    rows = index.long()[..., None].expand(-1, -1, -1, d)
    assert torch.equal(ko[:, :, :1], k.gather(2, rows)) and torch.equal(vo[:, :, :1], v.gather(2, rows))
    assert torch.equal(co[:, :, :1], com.gather(2, index.long()))
    assert bool((ko[:, :, 1:] == 0).all()) and bool((co[:, :, 1:] == 0).all())
