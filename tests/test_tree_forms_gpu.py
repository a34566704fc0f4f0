"""Every form of the tree step's kernels (head width, type, one or two tiles of nodes, the
launches apart or one workgroup per slice) and of the acceptance, against float64."""

from __future__ import annotations

import pytest
import torch

import serving_reference as ref
import test_tree_gpu as tree
from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]

WIDTHS = [16, 32, 64, 128, 256]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("n,count", [(7, 3), (32, 32), (33, 4), (64, 64)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_step_and_acceptance(d, dtype, n, count):
    """Few slices of 1541 keys: three launches, whole tiles and a part of one, several
    workgroups a slice.  The acceptance starts from the step's own lse, which is checked first."""
    from dilution import kernels

    b, h, length = 1, 2, 1541
    q, k, v, com = tree._make(10 * d + n, b, h, length, n, d, dtype, extra=1)
    parents = [tree._tree("chain" if count == n else "bushy", n, 1)]
    path = tree._paths(parents, count, 2)
    com[:, :, length:] = 0
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, parents, return_aux=True)
    tree._check_step(q, k, v, com, length, parents, out, aux["lse"])
    k0, v0, c0 = k.clone(), v.clone(), com.clone()
    kernels.dilution_tree_accept(q, k, v, com, length, aux["lse"], path)
    for j in range(h):
        want, rows = ref.accept_f64(q[0, j], k0[0, j], c0[0, j], length, aux["lse"][0, j], path[0])
        seen = torch.cat([k0[0, j, :length], k0[0, j][rows]])
        delta = ref.score_error(q[0, j], seen, d) + 2.0 ** -22 * aux["lse"][0, j].abs().max().item()
        # each bid's relative error (affinity, exp2), and the fp32 sum of the count + 1 terms
        bids = want.clone()
        bids[:length] -= c0[0, j, :length].double()
        bound = (2 * delta + 2.0 ** -20) * bids.abs() + (count + 1) * 2.0 ** -24 * want.abs() + 1e-12
        assert bool(((com[0, j, : length + count].double() - want).abs() <= bound).all()), j
        for cache, old in ((k, k0), (v, v0)):
            assert torch.equal(cache[0, j, length : length + count], old[0, j][rows])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_many_short_slices(d, dtype):
    """192 slices of 213 keys: one workgroup each, up to 32 nodes."""
    from dilution import kernels

    b, h, length, n = 12, 16, 213, 21
    q, k, v, com = tree._make(d, b, h, length, n, d, dtype)
    com[:, :, length:] = float("nan")
    parents = [tree._tree("bushy", n, i) for i in range(b)]
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, parents, return_aux=True)
    for i, j in ((0, 0), (5, 9), (11, 15)):
        at = (slice(i, i + 1), slice(j, j + 1))
        tree._check_step(q[at], k[at], v[at], com[at], length, [parents[i]], out[at], aux["lse"][at])
