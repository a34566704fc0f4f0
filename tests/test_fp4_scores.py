"""The bound on the 4-bit decode step's bids (tests/fp4_scores.py) holds for scores computed as the kernels do and
fails for planted mistakes, in a redone computation on the CPU."""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref
import fp4_scores as fs

WIDTHS = [16, 32, 64, 128, 256]
LENGTH = 400
VALUES = [1.9375, 1.0, 1.99999988079071044921875, 0.03125 + 2.0 ** -20]


def _ratios(d, part, spreads=fs.SPREADS):
    out = []
    for spread in spreads:
        q, codes, scales = fs.inputs(d, LENGTH, spread, seed=d + spread)
        k = ref.values(codes, scales)
        out.append(fs.worst(fs.computed_bids(q, k, part), *fs.bids(q, k)))
    return out


@pytest.mark.parametrize("d", WIDTHS)
def test_the_parts_are_the_query(d):
    """Whole numbers of -16 to 16 under each part's power, and less than 2^-39 of a block's largest left."""
    for spread in fs.SPREADS:
        q, _, _ = fs.inputs(d, LENGTH, spread, seed=d + spread)
        parts, n = fs.split(q), fs.blocks(d)
        top = q.double().view(*n).abs().amax(dim=1)
        _, power = torch.frexp(top)
        for i, x in enumerate(parts):
            digit = torch.ldexp(x.view(*n), 4 + 5 * i - power[:, None])
            assert (digit == digit.round()).all() and digit.abs().max() <= 16
        left = (q.double() - parts.sum(0)).view(*n).abs().amax(dim=1)
        assert (left <= 2.0 ** -39 * top).all()


@pytest.mark.parametrize("d", WIDTHS)
def test_right_scores_keep_the_bound(d):
    assert max(_ratios(d, lambda i, x: x)) <= 1


MISTAKES = {"the second four parts left out": lambda i, x: x if i < 4 else 0 * x}
for _p in range(fs.PARTS):
    MISTAKES[f"part {_p} left out"] = lambda i, x, p=_p: 0 * x if i == p else x
    MISTAKES[f"part {_p} at half its scale"] = lambda i, x, p=_p: x / 2 if i == p else x


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("mistake", MISTAKES)
def test_planted_mistakes_break_the_bound(d, mistake):
    assert max(_ratios(d, MISTAKES[mistake])) > 2


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("value", VALUES)
def test_a_lost_small_product_breaks_the_bound(d, value):
    q, codes, scales = fs.largest_sums(d, 300, value, seed=d)
    k = ref.values(codes, scales)
    want = fs.bids(q, k)
    assert fs.worst(fs.computed_bids(q, k), *want) <= 1
    small = k.abs() < k.abs().amax()
    assert small.sum() == 200
    assert fs.worst(fs.computed_bids(q, torch.where(small, 0.0, k)), *want) > 20
