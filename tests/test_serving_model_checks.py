"""The serving operators' host side, on the CPU: what the cache and the model check, keep and
refuse around the kernels."""

from __future__ import annotations

import pytest

from dilution.lm import Eviction


@pytest.mark.parametrize("limit,keep,first,recent", [(200, 100, 4, 48), (6, 5, 4, 1), (90, 50, 4, 23), (9, 4, 4, 0)])
def test_an_eviction_keeps_the_newest_by_default(limit, keep, first, recent):
    """Half of what the first ones leave, rounded up: the newest position stays where there is room."""
    rule = Eviction(limit=limit, keep=keep)
    assert (rule.first, rule.recent) == (first, recent)
    assert Eviction(limit=limit, keep=keep, recent=0).recent == 0
    assert Eviction(limit=limit, keep=keep, first=0).recent == (keep + 1) // 2


def test_an_eviction_has_room_for_the_first_ones():
    for bad in (dict(limit=10, keep=3), dict(limit=10, keep=3, first=4, recent=0), dict(limit=10, keep=8, recent=-1),
                dict(limit=10, keep=8, recent=5), dict(limit=10, keep=0, first=0)):
        with pytest.raises(ValueError, match="eviction"):
            Eviction(**bad)
