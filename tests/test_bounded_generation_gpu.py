"""Generations whose caches are bounded by an eviction: what their buffers hold, and when the
ones before are released."""

from __future__ import annotations

import weakref

import pytest
import torch

from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]


def _model():
    from dilution.lm import DilutionLM, LMConfig

    torch.manual_seed(3)
    return DilutionLM(LMConfig(vocab_size=300, n_layers=3, d_model=256, n_heads=4, prefill_chunk=64)).cuda().eval()


def _nothing(tokens):
    return torch.zeros(tokens.shape[0], 0, dtype=torch.long), []


@pytest.fixture
def evictions(monkeypatch):
    """(length before, capacity after) of every layer's evictions, and how many old buffers of
    this and the earlier layers live when a layer's turn comes."""
    from dilution import cache as dcache

    plain, seen, old = dcache.evict_cache, [], []

    def evict_cache(c, *args, **kw):
        if len(seen) % 3 == 0:
            old.clear()
        old.append(weakref.ref(c["k"]))
        alive = sum(r() is not None for r in old)
        before = c["len"]
        new = plain(c, *args, **kw)
        seen.append((before, new["len"], new["k"].shape[2], alive))
        return new

    monkeypatch.setattr(dcache, "evict_cache", evict_cache)
    return seen


@pytest.mark.parametrize("prompt,new", [(300, 60), (50, 100), (79, 30)])
def test_buffers_are_bounded_by_the_limit(evictions, prompt, new):
    """After an eviction the buffers hold the limit, whatever the prompt was; a layer's old buffer
    is gone before the next layer's turn; without drafts both generations give the same tokens."""
    from dilution.lm import Eviction

    model = _model()
    idx = torch.randint(0, 300, (2, prompt), generator=torch.Generator().manual_seed(8)).cuda()
    rule = Eviction(limit=80, keep=60, first=4, recent=16)
    plain = model.generate(idx, new, eviction=rule)
    assert plain.shape == (2, prompt + new) and torch.equal(plain[:, :prompt], idx)
    turns = len(evictions)
    assert turns >= 3 and turns % 3 == 0
    for before, after, capacity, alive in evictions:
        assert before >= 80 and after == 60 and 60 < capacity <= 80 and alive == 1
    drafted = model.generate_drafted(idx, new, _nothing, eviction=rule)
    assert len(evictions) == 2 * turns and torch.equal(drafted, plain)
    for before, after, capacity, alive in evictions[turns:]:
        assert before >= 80 and after == 60 and 60 < capacity <= 80 + 64 and alive == 1


def test_the_last_tokens_take_no_more_than_they_need(evictions):
    from dilution.lm import Eviction

    model = _model()
    idx = torch.randint(0, 300, (1, 100), generator=torch.Generator().manual_seed(9)).cuda()
    model.generate(idx, 5, eviction=Eviction(limit=90, keep=40, first=4, recent=8))
    assert [e[:3] for e in evictions] == [(100, 40, 44)] * 3


def test_drafts_over_bounded_caches(evictions):
    """Trees of the most nodes at every length up to the limit."""
    from dilution.lm import Eviction

    model = _model()
    idx = torch.randint(0, 300, (1, 60), generator=torch.Generator().manual_seed(10)).cuda()
    rule = Eviction(limit=70, keep=50, first=4, recent=16)

    def draft(tokens):                     # never right: token 299 is not picked below
        return torch.full((1, 63), 299), list(range(-1, 62))

    got = model.generate_drafted(idx, 45, draft, vocab_limit=299, eviction=rule)
    # 44 steps of one position from 60 on: the limit is reached before the 11th and, from 50 on,
    # 20 steps later; the next time would be before the 51st
    assert len(evictions) == 2 * 3 and all(e[0] == 70 and e[2] <= 70 + 64 for e in evictions)
    assert torch.equal(got, model.generate(idx, 45, vocab_limit=299, eviction=rule))


def test_evict_leaves_the_callers_caches():
    """DilutionLM.evict itself returns new caches and keeps the list that it was given."""
    from dilution.lm import Eviction

    model = _model()
    idx = torch.randint(0, 300, (1, 100), generator=torch.Generator().manual_seed(11)).cuda()
    _, caches = model.prefill(idx)
    given = list(caches)
    snap = [c["k"].clone() for c in caches]
    small = model.evict(caches, Eviction(limit=90, keep=50, first=4, recent=8), capacity=70)
    assert all(a is b for a, b in zip(caches, given)) and len(caches) == 3
    assert all(c["len"] == 100 and torch.equal(c["k"], s) for c, s in zip(caches, snap))
    assert all(c["len"] == 50 and c["k"].shape[2] == 70 for c in small)


def test_an_eviction_by_default_keeps_the_newest_rows():
    """The demand of a key grows with the rows that have seen it, so the newest hold the least of
    it: a window of them stays all the same."""
    from dilution.lm import Eviction

    model = _model()
    idx = torch.randint(0, 300, (2, 512), generator=torch.Generator().manual_seed(12)).cuda()
    _, caches = model.prefill(idx)
    small = model.evict(caches, Eviction(limit=512, keep=256))
    for old, new in zip(caches, small):
        for name in ("k", "v"):
            assert torch.equal(new[name][:, :, :4], old[name][:, :, :4])
            assert torch.equal(new[name][:, :, 256 - 126 :], old[name][:, :, 512 - 126 :])
