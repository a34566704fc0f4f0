"""The 4-bit decode step's bids and outputs on the GPU against float64, within the bound of its own arithmetic
(tests/fp4_scores.py, which test_fp4_scores.py shows to fail for planted mistakes)."""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref
import fp4_scores as fs
from dilution import kernels
from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]

TYPES = [torch.bfloat16, torch.float16, torch.float32]
WIDTHS = [16, 32, 64, 128, 256]


def _step(heads, dtype):
    """One step over heads of (q, codes, scales), no demand before: bids and outputs of each."""
    length, d = heads[0][1].shape[0], heads[0][0].shape[0]
    n = len(heads)
    g = torch.Generator().manual_seed(length + d)
    kc = kernels.Fp4Rows(*(torch.stack([x[i] for x in heads])[None].cuda() for i in (1, 2)))
    vc = kernels.Fp4Rows(*(x.cuda() for x in ref.quantise(torch.randn(1, n, length, d, generator=g))))
    com = torch.zeros(1, n, length, device="cuda")
    q = torch.stack([x[0] for x in heads])[None, :, None].to(dtype)
    out = kernels.dilution_decode_step_fp4(q.cuda(), kc, vc, com, length).cpu()
    kv, vv = ref.values(kc.codes.cpu(), kc.scales.cpu()), ref.values(vc.codes.cpu(), vc.scales.cpu())
    for i in range(n):
        p, rel = fs.bids(q[0, i, 0], kv[0, i])
        assert fs.worst(com[0, i], p, rel) <= 1
        want, _, spread, _ = ref.step_f64(q[0, i, 0], kv[0, i], vv[0, i], torch.zeros(length), length)
        bound = ref.out_bound(want, spread, dtype, rel.max().item(), length)
        assert ((out[0, i, 0].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [400, 9000])
@pytest.mark.parametrize("spread", fs.SPREADS)
def test_every_part_of_a_query_counts(d, dtype, length, spread):
    """Queries whose blocks hold elements 2^spread below their largest, which meets zeros only; one
    workgroup for a slice, and chunks."""
    _step([fs.inputs(d, length, spread, seed, dtype) for seed in (d + spread, length)], dtype)


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("value", [1.9375, 1.0, 1.99999988079071044921875, 0.03125 + 2.0 ** -20])
def test_one_small_product_among_the_largest(d, value):
    _step([fs.largest_sums(d, 300, value, seed) for seed in (d, d + 1)], torch.float32)


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("length", [400, 9000])
def test_small_queries_on_large_keys(d, dtype, length):
    """Queries down to subnormal elements, whose products with keys of powers up to 2^125 are of ordinary size."""
    _step([fs.small_query(d, length, top, d - top, dtype) for top in (-70, -85, -100, -106, -112, -119, -126, -135)], dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("length", [400, 9000])
def test_small_blocks_beside_ordinary_ones(d, length):
    _step([fs.small_query(d, length, top, d - top, beside=True) for top in (-85, -106, -119, -126, -135)], torch.float32)


@pytest.mark.parametrize("d", WIDTHS)
def test_a_block_that_is_no_number_meets_a_small_query(d):
    for length in (400, 9000):
        q, codes, scales = (x.cuda() for x in fs.small_query(d, length, -110, d))
        kc = kernels.Fp4Rows(codes[None, None].repeat(1, 2, 1, 1), scales[None, None].repeat(1, 2, 1, 1))
        kc.scales[0, 1, length // 2, -1] = 255
        vc = kernels.Fp4Rows(kc.codes.clone(), torch.full_like(kc.scales, 127))
        com = torch.zeros(1, 2, length, device="cuda")
        out = kernels.dilution_decode_step_fp4(q.expand(1, 2, 1, d), kc, vc, com, length)
        assert out[0, 0].isfinite().all() and com[0, 0].isfinite().all()
        assert out[0, 1].isnan().all() and com[0, 1].isnan().all()


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("length", [400, 9000])
def test_scores_at_the_end_of_fp32(d, dtype, length):
    """The type's largest value against a key of 1: the score is finite, its key takes the whole bid.  A row of
    equal scores as large divides it evenly."""
    q = torch.zeros(1, 2, 1, d, dtype=dtype)
    q[..., -1] = torch.finfo(dtype).max
    codes = torch.zeros(1, 2, length, d // 2, dtype=torch.uint8)
    codes[0, 0, :, -1] = 0x10                               # 0.5 in the last element
    codes[0, 0, 7, -1] = 0x20                               # 1
    codes[0, 1, :, -1] = 0x20
    kc = kernels.Fp4Rows(codes.cuda(), torch.full((1, 2, length, fs.blocks(d)[0]), 127, dtype=torch.uint8, device="cuda"))
    vc = kernels.Fp4Rows(*(x.cuda() for x in ref.quantise(torch.randn(1, 2, length, d, generator=torch.Generator().manual_seed(d)))))
    com = torch.zeros(1, 2, length, device="cuda")
    out = kernels.dilution_decode_step_fp4(q.cuda(), kc, vc, com, length).double().cpu()
    v = ref.values(*(x.cpu() for x in vc))[0]
    want = torch.zeros(length)
    want[7] = 1.0
    assert torch.equal(com[0, 0].cpu(), want)
    # shares of p / (p + eps), and their sum plus eps
    u = torch.finfo(dtype).eps / 2
    assert ((out[0, 0, 0] - v[0, 7] / (1 + 2e-9)).abs() <= (u + 2.0 ** -20) * v[0, 7].abs()).all()
    # even bids: every power is 1 and their sums are whole, so that only the division rounds (by a step at most)
    assert (com[0, 1].double().cpu() * length - 1).abs().max() <= 2 * fs.U
    # the mean: sums of length / 64 additions in a lane, 24 across lanes and waves
    mean = v[1].mean(0)
    assert ((out[0, 1, 0] - mean).abs() <= u * mean.abs() + 2.0 ** -14 * v[1].abs().mean(0)).all()
