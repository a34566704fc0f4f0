"""The tree step rounds to the outputs' type once, at its end: against float64, at inputs
where a rounding of the shares to 16 bits on the way is several times the bound."""

from __future__ import annotations

import pytest
import torch

import serving_reference as ref
from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]

BF16, F16 = torch.bfloat16, torch.float16


def _even_case(b, h, length, n, d, dtype):
    """Scores of at most some hundredths and demands between 0.5 and 1.5: many shares of one
    size, so the outputs are sums of values that cancel, and errors of the affinities are small."""
    g = torch.Generator().manual_seed(1000 * length + n)
    q = torch.randn(b, h, n, d, generator=g).mul(0.1).to(dtype).cuda()
    k = torch.randn(b, h, length + n, d, generator=g).mul(0.1).to(dtype).cuda()
    v = torch.randn(b, h, length + n, d, generator=g).to(dtype).cuda()
    com = (torch.rand(b, h, length + n, generator=g) + 0.5).cuda()
    return q, k, v, com


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,h,length,n,d", [
    (1, 2, 90, 8, 64),          # one workgroup for the whole step
    (1, 2, 1000, 8, 64),
    (1, 2, 1000, 40, 64),
    (1, 2, 700, 17, 16),
    (1, 2, 700, 50, 32),
    (1, 2, 1003, 13, 128),
    (1, 2, 600, 64, 128),
    (1, 2, 500, 20, 256),
    (1, 2, 500, 40, 256),
    (1, 1, 20000, 24, 64),
])
def test_shares_keep_their_bits(b, h, length, n, d, dtype):
    """Bound: half a step of the output's type once, and of the spread sum w |v| what fp32 work
    leaves: the bids' and the shares' two 16-bit parts (2^-16 each at most), the affinities'
    and lse's error (4 delta) and exp2, log2, rcp (2^-20); all of it twice, for the sum of
    share v and for the sum of the shares.  A lower part in fp16 is a multiple of 2^-24 of
    shares scaled by 2^14: an error of 2^-39 of each at most, under 2^-17 for shares over 2^-22."""
    from dilution import kernels

    q, k, v, com = _even_case(b, h, length, n, d, dtype)
    parents = [-1] + [max(i - 3, 0) for i in range(1, n)]
    out = kernels.dilution_tree_step(q, k, v, com, length, parents)
    u = torch.finfo(dtype).eps / 2
    for i in range(b):
        for j in range(h):
            want, lse, spread = ref.tree_f64(q[i, j], k[i, j], v[i, j], com[i, j], length, parents)
            delta = ref.score_error(q[i, j], k[i, j], d) + 2.0 ** -22 * max(1.0, lse.abs().max().item())
            share = 2 * 2.0 ** -16 + 4 * delta + 2.0 ** -20
            bound = u * want.abs() + 2 * share * spread + 1e-9
            err = (out[i, j].double() - want).abs()
            assert bool((err <= bound).all()), (i, j, (err / bound).max().item())
