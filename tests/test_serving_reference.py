"""The plain float64 forms that the drafted-token and eviction tests compare with:
pinned against the oracle's decode step, and mistakes planted in them are seen."""

from __future__ import annotations

import math

import pytest
import torch

import serving_reference as ref
from oracle import dilution_oracle as orc


def _inputs(seed, length, n, d=16):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(length + n, d, generator=g, dtype=torch.float64) for _ in range(3))
    com = torch.rand(length + n, generator=g, dtype=torch.float64) * 2
    com[length:] = 0
    return q[length:], k, v, com


def _decode_chain(q, k, v, com, length, chain):
    """The oracle's decode step token after token down one chain."""
    kk, vv = k[:length].clone(), v[:length].clone()
    com = com[:length].clone()
    for step, node in enumerate(chain):
        kk = torch.cat([kk, k[length + node][None]])
        vv = torch.cat([vv, v[length + node][None]])
        com = torch.cat([com, torch.zeros(1, dtype=com.dtype)])
        y, com_new = orc.decode_step(q[node].view(1, 1, 1, -1), kk[None, None], vv[None, None], com[None, None],
                                     length + step + 1)
        com = com_new.reshape(-1)
    return y.reshape(-1), com


PARENTS = [-1, 0, 0, 1, 3, 2, -1, 6, 4]


@pytest.mark.parametrize("length", [0, 1, 37])
def test_tree_nodes_are_decode_steps_down_their_chains(length):
    q, k, v, com = _inputs(1, length, len(PARENTS))
    out, lse, spread = ref.tree_f64(q, k, v, com, length, PARENTS)
    for i in range(len(PARENTS)):
        chain = ref.chain_of(PARENTS, i)
        y, after = _decode_chain(q, k, v, com, length, chain)
        assert (out[i] - y).abs().max() < 1e-12
        assert bool((spread[i] >= out[i].abs() - 1e-12).all())
        new, rows = ref.accept_f64(q, k, com, length, lse, chain)
        assert (new - after).abs().max() < 1e-12
        assert rows.tolist() == [length + c for c in chain]


def test_absent_nodes_take_those_below_with_them():
    parents = [-1, -2, 1, 0, 9, -7]
    assert [ref.chain_of(parents, i) for i in range(6)] == [[0], None, None, [0, 3], None, None]


def test_planted_mistakes_are_seen():
    """A tree that lets a node see a sibling, or drops an ancestor's demand, is off
    by more than the bound of bf16 outputs."""
    q, k, v, com = _inputs(2, 24, 4)
    parents = [-1, 0, 0, 2]
    out, _, spread = ref.tree_f64(q, k, v, com, 24, parents)
    bound = ref.out_bound(out, spread, torch.bfloat16, 0.0)
    sibling, _, _ = ref.tree_f64(q, k, v, com, 24, [-1, 0, 1, 2])
    assert bool(((sibling - out).abs() > bound).any())
    dropped = out.clone()
    dropped[3] = ref.tree_f64(q[[3]], torch.cat([k[:24], k[[27]]]), torch.cat([v[:24], v[[27]]]), com, 24, [-1])[0][0]
    assert bool(((dropped - out).abs() > bound).any())


def test_eviction_order():
    nan = math.nan
    com = torch.tensor([5.0, 1.0, 0.0, -0.0, 2.0, 2.0, nan, 2.0, 0.0, 9.0])
    assert ref.evict_f64(com, 10, 5, 0, 0) == [0, 4, 5, 6, 9]
    assert ref.evict_f64(com, 10, 6, 1, 2) == [0, 4, 5, 6, 8, 9]
    assert ref.evict_f64(com, 10, 9, 0, 1) == [0, 1, 2, 3, 4, 5, 6, 7, 9]
