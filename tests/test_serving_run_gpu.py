"""The serving operators together, as a generation uses them: prefill, eviction, tree
steps, acceptance and decode steps on one cache, and the language model on them."""

from __future__ import annotations

import math

import pytest
import torch

import serving_reference as ref
from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]


def _rows(g, b, h, n, d, dtype):
    return [torch.randn(b, h, n, d, generator=g).to(dtype).cuda() for _ in range(3)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_generation_on_one_cache(dtype):
    """Every output and the demand against float64 forms that run on the cache's own rows; the
    demand they start from is the kernels' own at each step, so the bounds do not add up."""
    from dilution import cache as dcache

    b, h, d, prompt = 2, 2, 64, 400
    g = torch.Generator().manual_seed(0)
    q, k, v = _rows(g, b, h, prompt, d, dtype)
    _, c = dcache.begin_cache(q, k, v, capacity=prompt + 40, chunk=128)
    for turn in range(3):
        old = {x: c[x].clone() for x in ("k", "v", "committed")}
        keep = c["len"] - 60
        before = c["len"]
        c = dcache.evict_cache(c, keep, first=2, recent=20, capacity=keep + 40)
        assert c["len"] == keep and c["k"].shape[2] == keep + 40
        for i in range(b):
            for j in range(h):
                rows = ref.evict_f64(old["committed"][i, j].cpu(), before, keep, 2, 20)
                assert torch.equal(c["k"][i, j, :keep], old["k"][i, j, rows])
                assert torch.equal(c["committed"][i, j, :keep], old["committed"][i, j, rows])
        # a tree, twice: the first is thrown away
        parents = [-1, 0, 0, 1, 3, 2, 1]
        for attempt in range(2):
            q, k, v = _rows(g, b, h, 7, d, dtype)
            y, draft = dcache.tree_step(q, k, v, c, parents)
            assert c["len"] == keep and bool((c["committed"][:, :, keep:] == 0).all())
        for i in range(b):
            for j in range(h):
                want, lse, spread = ref.tree_f64(q[i, j], c["k"][i, j], c["v"][i, j], c["committed"][i, j], keep, parents)
                delta = ref.score_error(q[i, j], c["k"][i, j, : keep + 7], d) + 2.0 ** -22 * 10
                err = (y[i, j].double() - want).abs()
                assert bool((err <= ref.out_bound(want, spread, dtype, delta)).all()), (turn, i, j)
        snap = {x: c[x].clone() for x in ("k", "committed")}
        path = [[0, 1, 3], [0, 2, 5]]
        assert dcache.accept_tree(c, draft, path) == keep + 3 == c["len"]
        for i in range(b):
            for j in range(h):
                want, rows = ref.accept_f64(q[i, j], snap["k"][i, j], snap["committed"][i, j], keep, draft["lse"][i, j], path[i])
                assert (c["committed"][i, j, : keep + 3] - want).abs().max().item() < 1e-5
                assert torch.equal(c["k"][i, j, keep : keep + 3], snap["k"][i, j][rows])
        assert bool((c["committed"][:, :, keep + 3 :] == 0).all())
        with pytest.raises(ValueError, match="moved on"):
            dcache.accept_tree(c, draft, [0])
        # and a plain decode step over it
        q1, k1, v1 = _rows(g, b, h, 1, d, dtype)
        com = c["committed"].clone()
        y1 = dcache.step_cache(q1, k1, v1, c)
        n = c["len"]
        for i in range(b):
            for j in range(h):
                want, _, spread = ref.tree_f64(q1[i, j], c["k"][i, j, :n], c["v"][i, j, :n], com[i, j], n - 1, [-1])
                delta = ref.score_error(q1[i, j], c["k"][i, j, :n], d) + 2.0 ** -22 * 10
                assert bool(((y1[i, j].double() - want).abs() <= ref.out_bound(want, spread, dtype, delta)).all())


def _model(dtype, **kw):
    from dilution.lm import DilutionLM, LMConfig

    torch.manual_seed(3)
    cfg = LMConfig(vocab_size=300, n_layers=3, d_model=256, n_heads=4, prefill_chunk=64, **kw)
    return DilutionLM(cfg).cuda().to(dtype).eval()


def test_model_tree_step_is_its_decode_steps():
    """Logits of a tree's nodes against decoding each path token by token, in fp32 (the paths
    differ by fp32 rounding only), and the caches after the acceptance."""
    model = _model(torch.float32)
    g = torch.Generator().manual_seed(1)
    idx = torch.randint(0, 300, (2, 90), generator=g).cuda()
    tree = torch.randint(0, 300, (2, 6), generator=g).cuda()
    parents = [-1, 0, 0, 1, 3, 2]
    _, caches = model.prefill(idx, capacity=110)
    logits, drafts = model.tree_step(tree, parents, caches)
    for leaf in (4, 5):
        chain = ref.chain_of(parents, leaf)
        _, plain = model.prefill(idx, capacity=110)
        for node in chain:
            want = model.decode_step(tree[:, node : node + 1], plain)
            assert (logits[:, node] - want[:, 0]).abs().max().item() < 2e-4 * want.abs().max().item() + 1e-5
    assert model.accept_tree(caches, drafts, ref.chain_of(parents, 5)) == 93
    for a, b in zip(caches, plain):
        assert a["len"] == b["len"] == 93
        assert (a["k"][:, :, :93] - b["k"][:, :, :93]).abs().max().item() < 1e-3
        assert (a["committed"] - b["committed"]).abs().max().item() < 1e-3
    nxt = torch.randint(0, 300, (2, 1), generator=g).cuda()
    x, y = model.decode_step(nxt, caches), model.decode_step(nxt, plain)
    assert (x - y).abs().max().item() < 2e-4 * y.abs().max().item() + 1e-5


@pytest.mark.parametrize("quality", ["right", "wrong", "mixed", "none"])
def test_drafted_generation_gives_the_greedy_tokens(quality):
    model = _model(torch.float32)
    g = torch.Generator().manual_seed(2)
    idx = torch.randint(0, 300, (1, 40), generator=g).cuda()
    want = model.generate(idx, 24, vocab_limit=290)
    calls = []

    def draft(tokens):
        calls.append(tokens.shape[1])
        t = tokens.shape[1]
        ahead = [int(x) for x in want[0, t : t + 3]]
        if quality == "none":
            return torch.zeros(1, 0, dtype=torch.long), []
        if quality == "wrong" or not ahead:
            return torch.full((1, 2), 299), [-1, 0]
        if quality == "mixed":             # a wrong sibling first, then the right token
            return torch.tensor([[299] + ahead]), [-1, -1] + list(range(1, len(ahead)))
        return torch.tensor([ahead]), list(range(-1, len(ahead) - 1))

    got = model.generate_drafted(idx, 24, draft, vocab_limit=290)
    assert torch.equal(got, want)
    assert len(calls) <= 8 if quality in ("right", "mixed") else len(calls) == 23


def test_drafted_batch_keeps_its_sequences_in_step():
    model = _model(torch.float32)
    idx = torch.randint(0, 300, (3, 33), generator=torch.Generator().manual_seed(5)).cuda()
    want = model.generate(idx, 15)

    def draft(tokens):
        t = tokens.shape[1]
        ahead = want[:, t : t + 4].clone()
        if ahead.shape[1] > 1:
            ahead[1, 1] = 0                # the second sequence's draft is wrong from its second token
        return ahead, list(range(-1, ahead.shape[1] - 1))

    assert torch.equal(model.generate_drafted(idx, 15, draft), want)


def test_generation_with_bounded_caches():
    """An eviction that never comes changes nothing; one that does keeps the caches bounded."""
    from dilution.lm import Eviction

    model = _model(torch.bfloat16)
    idx = torch.randint(0, 300, (2, 100), generator=torch.Generator().manual_seed(6)).cuda()
    plain = model.generate(idx, 12)
    assert torch.equal(model.generate(idx, 12, eviction=Eviction(limit=4000, keep=2000)), plain)
    short = model.generate(idx, 40, eviction=Eviction(limit=80, keep=60, first=4, recent=16))
    assert short.shape == (2, 140) and torch.equal(short[:, :100], idx)
    none = lambda tokens: (torch.zeros(2, 0, dtype=torch.long), [])  # noqa: E731
    drafted = model.generate_drafted(idx, 40, none, eviction=Eviction(limit=80, keep=60, first=4, recent=16))
    assert drafted.shape == (2, 140)
    _, caches = model.prefill(idx)
    small = model.evict(caches, Eviction(limit=90, keep=50), capacity=70)
    assert all(c["len"] == 50 and c["k"].shape[2] == 70 for c in small)
    assert all(math.isfinite(c["committed"].sum().item()) for c in small)
