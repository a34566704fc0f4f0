"""The serving operators' host side, on the CPU: what the cache and the model check, keep and
refuse around the kernels."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from dilution import cache, kernels
from dilution.lm import DilutionLM, Eviction, LMConfig


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


def _state(b=2, h=3, cap=40, n=4, d=64):
    q = torch.zeros(b, h, n, d, dtype=torch.bfloat16)
    k = torch.zeros(b, h, cap, d, dtype=torch.bfloat16)
    return q, k, k.clone(), torch.zeros(b, h, cap)


def test_host_node_numbers_are_whole_and_checked():
    """Numbers that are not whole are refused, not cut; so are the shapes that no tree has."""
    q, k, v, com = _state()
    lse = torch.zeros(2, 3, 4)
    for bad in ([-1, 0.0, 1.0, 5.7], [-1.0, 0.5, 1.0, 2.0], np.array([-1.0, 0, 1, 2]), [True, False, False, False]):
        with pytest.raises(ValueError, match="parents must be int32 or int64"):
            kernels.dilution_tree_step(q, k, v, com, 36, bad)
    for bad in ([0.0, 1.5], np.array([0.5]), [False, True]):
        with pytest.raises(ValueError, match="path must be int32 or int64"):
            kernels.dilution_tree_accept(q, k, v, com, 36, lse, bad)
    for bad in (0, torch.tensor(0), np.int64(0), [[[0, 1]]], torch.zeros(1, 1, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="path"):
            kernels.dilution_tree_accept(q, k, v, com, 36, lse, bad)
    for bad in (0, torch.tensor(-1), [[[-1, 0, 1, 2]]]):
        with pytest.raises(ValueError, match="parents"):
            kernels.dilution_tree_step(q, k, v, com, 36, bad)
    # what is whole passes these checks (and stops at the tensors, which are on the CPU)
    for good in ([-1, 0, 1, 2], (-1, 0, 1, -2), np.array([-1, 0, 1, 2]), np.array([-1, 0, 1, 2], dtype=np.int32),
                 np.array([-1, 0, 1, 2], dtype=np.int16),
                 torch.tensor([[-1, 0, 1, 2]] * 2)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            kernels.dilution_tree_step(q, k, v, com, 36, good)
    for good in ([], [[], []], [0, 3], np.array([1, 2]), np.array([0, 3], dtype=np.uint32), np.array([2], dtype=np.uint8)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            kernels.dilution_tree_accept(q, k, v, com, 36, lse, good)


def _model(**kw):
    return DilutionLM(LMConfig(vocab_size=32, n_layers=3, d_model=64, n_heads=4, **kw))


def test_a_model_step_converts_its_tree_once(monkeypatch):
    """Every layer gets the same int32 tensor; a tree that is refused reaches none."""
    model, seen = _model(), []

    def tree_step(q, k, v, cache, parents):
        seen.append(parents)
        return q, {}

    monkeypatch.setattr(cache, "tree_step", tree_step)
    tokens = torch.zeros(1, 4, dtype=torch.long)
    model.tree_step(tokens, [-1, 0, 1, -2], [{}] * 3)
    assert len(seen) == 3 and all(p is seen[0] for p in seen)
    assert seen[0].dtype == torch.int32 and seen[0].tolist() == [-1, 0, 1, -2]
    with pytest.raises(ValueError, match="parent"):
        model.tree_step(tokens, [-1, 0, 2, 1], [{}] * 3)
    assert len(seen) == 3


@pytest.fixture
def on_cpu(monkeypatch):
    """The kernels' calls replaced: only what the cache dict and the model do around them runs."""
    monkeypatch.setattr(kernels, "dilution_tree_step", lambda q, k, v, com, t, parents, return_aux: (q, {"lse": None}))
    monkeypatch.setattr(kernels, "dilution_tree_accept", lambda q, k, v, com, t, lse, path: t + len(path))


def _cache(length=30):
    _, k, v, com = _state()
    return {"k": k, "v": v, "len": length, "committed": com}


def _draft(c, n=4, **kw):
    q = torch.ones(2, 3, n, 64, dtype=torch.bfloat16)
    return cache.tree_step(q, kw.get("k", q), kw.get("v", q), c, list(range(-1, n - 1)))[1]


def test_only_the_last_draft_is_accepted(on_cpu):
    """A second tree step has overwritten the first one's rows, at the same length."""
    c = _cache()
    first, second = _draft(c), _draft(c)
    with pytest.raises(ValueError, match="moved on"):
        cache.accept_tree(c, first, [0])
    assert c["len"] == 30
    with pytest.raises(ValueError, match="moved on"):      # of another cache, as long
        cache.accept_tree(_cache(), second, [0])
    assert cache.accept_tree(c, second, []) == 30          # nothing taken, nothing moved
    assert cache.accept_tree(c, second, [0, 1]) == 32
    for length in (32, 30):
        c["len"] = length
        with pytest.raises(ValueError, match="moved on"):
            cache.accept_tree(c, second, [0])


def test_a_decode_step_takes_the_draft_away(on_cpu):
    c = _cache()
    draft = _draft(c)
    one = torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16)
    cache.append_kv(c, one, one)
    c["len"] = 30                                          # as a program that takes the token back
    with pytest.raises(ValueError, match="moved on"):
        cache.accept_tree(c, draft, [0])


def test_a_refused_tree_step_leaves_the_draft_before_it(on_cpu):
    c = _cache()
    draft = _draft(c)
    rows = [c[x].clone() for x in ("k", "v")]
    q = torch.full((2, 3, 4, 64), 7.0, dtype=torch.bfloat16)
    for args, kind in (((q, q, q, c, [-1, 0, 2, 1]), "parent"), ((q, q, q, c, [-1, 0, 1]), "parents"),
                       ((q, q, q, c, torch.zeros(3, 4, dtype=torch.int32)), "parent"),
                       ((q, q, q, c, torch.zeros(3, 4, dtype=torch.int32) - 1), "parents"),
                       ((q, q[:, :, :1], q, c, [-1] * 4), "one shape"), ((q, q, q[:1], c, [-1] * 4), "one shape"),
                       ((q[:1], q[:1], q[:1], c, [-1] * 4), "cache"), ((q[..., :32],) * 3 + (c, [-1] * 4), "cache"),
                       ((q.float(), q, q, c, [-1] * 4), "dtype"), ((q[:, :, :0],) * 3 + (c, []), "1 to 64"),
                       ((q.repeat(1, 1, 3, 1),) * 3 + (c, [-1] * 12), "capacity"),
                       ((q[0], q[0], q[0], c, [-1] * 3), "B, H, N, D")):
        with pytest.raises(ValueError, match=kind):
            cache.tree_step(*args)
    for x, old in zip(("k", "v"), rows):
        assert torch.equal(c[x], old)
    big = {"k": torch.zeros(2, 3, 99, 64, dtype=torch.bfloat16), "len": 0}
    with pytest.raises(ValueError, match="1 to 64"):
        cache.tree_step(*(q.repeat(1, 1, 17, 1),) * 3, big, [-1] * 68)
    assert cache.accept_tree(c, draft, [0, 1]) == 32


def test_a_model_accepts_in_every_layer_or_none(on_cpu):
    model = _model()
    caches = [_cache() for _ in range(3)]
    drafts = [_draft(c) for c in caches]
    with pytest.raises(ValueError, match="drafts"):
        model.accept_tree(caches, drafts[:2], [0])
    last = _draft(caches[2])
    with pytest.raises(ValueError, match="moved on"):
        model.accept_tree(caches, drafts, [0])
    assert [c["len"] for c in caches] == [30] * 3
    assert model.accept_tree(caches, drafts[:2] + [last], [0, 1]) == 32
