"""The tree step and the acceptance of drafted tokens on the GPU, against the plain
float64 forms of serving_reference (elementwise bounds derived there)."""

from __future__ import annotations

import math

import pytest
import torch

import serving_reference as ref
from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _make(seed, b, h, length, n, d, dtype, extra=0, scale=1.0, strided=True):
    g = torch.Generator().manual_seed(seed)
    cap = length + n + extra
    q = torch.randn(b, n, h * d, generator=g).mul(scale).to(dtype).cuda().view(b, n, h, d).transpose(1, 2)
    if not strided:
        q = q.contiguous()
    k = torch.randn(b, h, cap, d, generator=g).mul(scale).to(dtype).cuda()
    v = torch.randn(b, h, cap, d, generator=g).to(dtype).cuda()
    com = torch.zeros(b, h, cap)
    com[:, :, :length] = torch.rand(b, h, length, generator=g) * 3 * (torch.rand(b, h, length, generator=g) > 0.1)
    return q, k, v, com.cuda()


def _tree(kind, n, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "flat":
        return [-1] + [0] * (n - 1)
    if kind == "roots":
        return [-1] * n
    return [-1] + [int(torch.randint(max(-1, i - 7), i, (1,), generator=g)) for i in range(1, n)]


def _check_step(q, k, v, com, length, parents, out, lse):
    """parents: one list per batch."""
    b, h, n, d = q.shape
    for i in range(b):
        for j in range(h):
            want, wl, spread = ref.tree_f64(q[i, j], k[i, j], v[i, j], com[i, j], length, parents[i])
            here = torch.isfinite(wl)
            assert torch.equal(here.cpu(), torch.isfinite(lse[i, j]).cpu()) and bool((lse[i, j][~here.to(lse.device)] == math.inf).all())
            if not bool(here.any()):
                assert bool((out[i, j] == 0).all())
                continue
            rows = length + here.nonzero()[:, 0]
            delta = ref.score_error(q[i, j][here], torch.cat([k[i, j, :length], k[i, j][rows]]), d) + 2.0 ** -22 * max(
                1.0, wl[here].abs().max().item())
            # lse: the affinities' error, and a log2 of a sum of up to 2^17 terms
            assert (lse[i, j].double() - wl)[here].abs().max().item() <= delta + 2.0 ** -20, (i, j)
            err = (out[i, j].double() - want).abs()
            bound = ref.out_bound(want, spread, out.dtype, delta)
            assert bool((err <= bound).all()), (i, j, (err / bound).max().item(), err.max().item())
            assert bool((out[i, j][~here] == 0).all())


SHAPES = [
    # b, h, length, n, d, dtype, kind
    (1, 1, 0, 1, 64, BF16, "chain"),
    (1, 2, 0, 64, 64, BF16, "bushy"),
    (1, 2, 1, 1, 64, BF16, "chain"),
    (2, 3, 1, 2, 16, F32, "flat"),
    (1, 2, 31, 31, 32, BF16, "bushy"),
    (2, 1, 32, 32, 64, F16, "bushy"),
    (1, 3, 33, 33, 64, BF16, "bushy"),
    (1, 2, 127, 63, 128, BF16, "chain"),
    (1, 2, 255, 64, 64, BF16, "roots"),
    (2, 2, 256, 8, 64, BF16, "bushy"),
    (3, 5, 1003, 13, 128, F16, "bushy"),
    (1, 4, 1000, 8, 64, F32, "bushy"),
    (2, 2, 777, 40, 32, F32, "chain"),
    (1, 2, 515, 64, 128, F32, "bushy"),
    (1, 2, 700, 33, 256, BF16, "bushy"),
    (1, 2, 129, 64, 256, F16, "chain"),
    (1, 2, 300, 17, 256, F32, "bushy"),
    (1, 3, 600, 64, 16, BF16, "bushy"),
    (2, 3, 5000, 5, 64, BF16, "chain"),
    (1, 2, 20001, 24, 64, BF16, "bushy"),
    (1, 1, 9000, 64, 32, F16, "bushy"),
    (4, 16, 2500, 16, 64, BF16, "bushy"),
]


@pytest.mark.parametrize("b,h,length,n,d,dtype,kind", SHAPES)
def test_step_matches_float64(b, h, length, n, d, dtype, kind):
    from dilution import kernels

    q, k, v, com = _make(length + n, b, h, length, n, d, dtype, extra=3)
    # what lies behind the drafted rows, and the demand of the drafted positions, is not read
    k[:, :, length + n :] = v[:, :, length + n :] = float("nan")
    com[:, :, length:] = float("nan")
    before = [t.clone() for t in (k, v, com)]
    parents = [_tree(kind, n, 10 * i) for i in range(b)]
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, parents, return_aux=True)
    assert out.dtype == dtype and out.shape == q.shape and aux["lse"].dtype == F32
    _check_step(q, k, v, com, length, parents, out, aux["lse"])
    for t, s in zip((k, v, com), before):
        assert torch.equal(t.view(torch.uint8), s.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("length", [0, 70, 4097])
def test_absent_nodes_and_their_garbage_count_for_nothing(dtype, length):
    """Padded trees: absent nodes (and those below) hold NaN and infinities in q, k and v."""
    from dilution import kernels

    b, h, n, d = 2, 2, 37, 64
    q, k, v, com = _make(5, b, h, length, n, d, dtype)
    parents = [_tree("bushy", n, 3), _tree("bushy", n, 4)]
    parents[0][20:] = [-2] * 17
    parents[1][5] = -2
    for i, tree in enumerate(parents):
        for node in range(n):
            if ref.chain_of(tree, node) is None:
                q[i, :, node] = float("nan") if node % 2 else float("inf")
                k[i, :, length + node] = float("inf") if node % 2 else float("nan")
                v[i, :, length + node] = float("nan")
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, torch.tensor(parents), return_aux=True)
    _check_step(q, k, v, com, length, parents, out, aux["lse"])


def test_wild_device_parents_are_absent_nodes():
    from dilution import kernels

    n = 12
    q, k, v, com = _make(6, 1, 2, 50, n, 64, BF16)
    wild = [-1, 0, 7, 2147483647, -2147483648, 1, 5, 4, 8, 11, 6, 10]
    for dt in (torch.int32, torch.int64):
        out, aux = kernels.dilution_tree_step(q, k, v, com, 50, torch.tensor(wild, dtype=dt).cuda(), return_aux=True)
        _check_step(q, k, v, com, 50, [wild], out, aux["lse"])
    big = torch.tensor(wild).cuda()
    big[3] = 4294967295          # -1 in its low 32 bits
    big[4] = -4294967296
    again = kernels.dilution_tree_step(q, k, v, com, 50, big)
    assert torch.equal(again, out)


@pytest.mark.parametrize("length,n", [(333, 40), (333, 30), (100, 30), (0, 20)])
@pytest.mark.parametrize("bad", ["nan_q", "inf_q", "nan_v", "nan_k"])
def test_a_broken_branch_stays_its_own(bad, length, n):
    """A node that holds NaN spoils itself and the nodes below it, and no bit of the others."""
    from dilution import kernels

    q, k, v, com = _make(7, 1, 2, length, n, 64, BF16, strided=False)
    parents = _tree("bushy", n, 9)
    clean, aux = kernels.dilution_tree_step(q, k, v, com, length, parents, return_aux=True)
    node = 6
    if bad.endswith("q"):
        q[:, :, node] = float(bad[:3])
    else:
        {"k": k, "v": v}[bad[-1]][:, :, length + node] = float("nan")
    out, aux2 = kernels.dilution_tree_step(q, k, v, com, length, parents, return_aux=True)
    hit = [node in ref.chain_of(parents, i) for i in range(n)]
    assert any(hit) and not all(hit)
    for i in range(n):
        if hit[i]:
            assert bool(torch.isnan(out[:, :, i]).all()), i
        else:
            assert torch.equal(out[:, :, i], clean[:, :, i]) and torch.equal(aux2["lse"][:, :, i], aux["lse"][:, :, i]), i


def test_nan_and_inf_in_the_cache_reach_every_node():
    from dilution import kernels

    for where in ("k", "v", "committed"):
        q, k, v, com = _make(8, 1, 2, 200, 9, 64, BF16)
        {"k": k, "v": v, "committed": com}[where][:, 1, 77] = float("nan")
        out = kernels.dilution_tree_step(q, k, v, com, 200, _tree("bushy", 9, 1))
        assert bool(torch.isnan(out[:, 1]).all()) and bool(torch.isfinite(out[:, 0]).all()), where


@pytest.mark.parametrize("dtype,scale", [(BF16, 6.0), (F32, 6.0), (F16, 0.01), (BF16, 0.0)])
def test_peaked_and_flat_rows(dtype, scale):
    """Scores of hundreds (almost all bids 0) and none at all (uniform bids)."""
    from dilution import kernels

    length, n, d = 1500, 20, 64
    q, k, v, com = _make(11, 1, 2, length, n, d, dtype, scale=scale)
    parents = [_tree("bushy", n, 2)]
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, parents[0], return_aux=True)
    _check_step(q, k, v, com, length, parents, out, aux["lse"])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_chain_is_a_prefill_chunk_and_decode_steps(dtype):
    """The same rows by the other paths of the library; each side is within its bound of float64,
    so they are within the sum."""
    from dilution import kernels

    b, h, length, n, d = 2, 4, 600, 12, 64
    q, k, v, com = _make(12, b, h, length, n, d, dtype, strided=False)
    com[:, :, length:] = 0
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, _tree("chain", n, 0), return_aux=True)
    c1, rows = com.clone(), []
    for i in range(n):
        rows.append(kernels.dilution_decode_step(q[:, :, i : i + 1].contiguous(), k, v, c1, length + i + 1))
    dec = torch.cat(rows, dim=2)
    tol = 3e-2 if dtype == BF16 else 2e-5            # two bf16 outputs of O(1), or fp32 sums
    assert (out.double() - dec.double()).abs().max().item() <= tol
    c2 = com.clone()
    pre = kernels.dilution_prefill_chunk(q, k, v, c2, length, dot_precision="bf16" if dtype == BF16 else "ieee")
    assert (out.double() - pre.double()).abs().max().item() <= tol
    assert kernels.dilution_tree_accept(q, k, v, com, length, aux["lse"], list(range(n))) == length + n
    assert (com - c1).abs().max().item() <= 1e-4 and (com - c2).abs().max().item() <= 1e-4


def test_trees_given_in_every_form():
    from dilution import kernels

    b, n = 3, 10
    q, k, v, com = _make(13, b, 2, 90, n, 32, BF16)
    tree = _tree("bushy", n, 5)
    forms = [tree, tuple(tree), [tree] * b, torch.tensor(tree), torch.tensor([tree] * b), torch.tensor(tree).cuda(),
             torch.tensor([tree] * b, dtype=torch.int32).cuda(),
             torch.tensor([tree] * b, dtype=torch.int32).t().contiguous().t().cuda()]
    outs = [kernels.dilution_tree_step(q, k, v, com, 90, f) for f in forms]
    for o in outs[1:]:
        assert torch.equal(o, outs[0])
    assert outs[0].stride() == q.stride()             # (B, N, H, D) memory, as the queries
    assert torch.equal(kernels.dilution_tree_step(q.contiguous(), k, v, com, 90, tree), outs[0])


def test_empty_batch():
    from dilution import kernels

    q, k, v, com = _make(14, 1, 2, 20, 4, 32, BF16)
    out, aux = kernels.dilution_tree_step(q[:0], k[:0], v[:0], com[:0], 20, [-1, 0, 0, 0], return_aux=True)
    assert out.shape == (0, 2, 4, 32)
    assert kernels.dilution_tree_accept(q[:0], k[:0], v[:0], com[:0], 20, aux["lse"], [0, 1]) == 22


@pytest.mark.parametrize("b,h,length,n,d,dtype", [
    (48, 16, 1501, 20, 64, BF16),          # as many slices as the GPU holds: a workgroup each
    (16, 12, 255, 32, 64, BF16),           # 192 slices of few keys
    (16, 12, 257, 32, 64, F16),            # and of more
    (32, 16, 900, 9, 128, F16),
    (48, 16, 333, 17, 32, F32),
    (24, 16, 1000, 3, 64, F32),
    (16, 16, 500, 12, 256, BF16),
    (16, 16, 300, 5, 256, F32),
    (30, 30, 700, 8, 16, BF16),
    (48, 16, 600, 40, 64, BF16),           # two node tiles: never one workgroup
])
def test_many_slices_match_float64(b, h, length, n, d, dtype):
    from dilution import kernels

    q, k, v, com = _make(length, b, h, length, n, d, dtype, extra=1)
    com[:, :, length:] = float("nan")
    k[:, :, length + n :] = v[:, :, length + n :] = float("nan")
    parents = [_tree("bushy", n, i) for i in range(b)]
    parents[1] = parents[1][: n - 1] + [-2]
    k[1, :, length + n - 1] = v[1, :, length + n - 1] = q[1, :, n - 1] = float("nan")
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, parents, return_aux=True)
    for i, j in ((0, 0), (1, 1), (b // 2, h - 1), (b - 1, h - 1)):
        one = slice(i, i + 1)
        _check_step(q[one, j : j + 1], k[one, j : j + 1], v[one, j : j + 1], com[one, j : j + 1], length, [parents[i]],
                    out[one, j : j + 1], aux["lse"][one, j : j + 1])
    again = kernels.dilution_tree_step(q, k, v, com, length, parents)
    assert torch.equal(again, out)


# ---------------------------------------------------------------------------
# acceptance


def _paths(parents, count, seed):
    """A chain of up to `count` nodes from a root of every tree, all equally long."""
    g = torch.Generator().manual_seed(seed)
    chains = []
    for tree in parents:
        full = [ref.chain_of(tree, i) for i in range(len(tree))]
        full = [c for c in full if c is not None and len(c) >= count]
        chains.append(full[int(torch.randint(len(full), (1,), generator=g))][:count])
    return chains


ACCEPTS = [
    # b, h, length, n, d, dtype, kind, count
    (1, 1, 0, 1, 64, BF16, "chain", 1),
    (1, 2, 0, 9, 64, BF16, "chain", 9),
    (2, 2, 1, 5, 16, F32, "chain", 3),
    (2, 3, 33, 20, 64, BF16, "bushy", 3),
    (1, 2, 255, 64, 64, F16, "chain", 64),
    (1, 2, 256, 33, 128, BF16, "chain", 33),
    (2, 2, 257, 30, 256, BF16, "bushy", 3),
    (1, 2, 100, 64, 256, F32, "chain", 64),
    (3, 5, 5003, 13, 128, F16, "bushy", 2),
    (2, 12, 9001, 24, 32, F32, "bushy", 4),
    (4, 16, 2500, 16, 64, BF16, "bushy", 3),
]


@pytest.mark.parametrize("b,h,length,n,d,dtype,kind,count", ACCEPTS)
def test_accept_matches_float64(b, h, length, n, d, dtype, kind, count):
    from dilution import kernels

    q, k, v, com = _make(length + n + 1, b, h, length, n, d, dtype, extra=2)
    parents = [_tree(kind, n, 7 * i + 1) for i in range(b)]
    path = _paths(parents, count, 3)
    _, aux = kernels.dilution_tree_step(q, k, v, com, length, parents, return_aux=True)
    k0, v0, c0 = k.clone(), v.clone(), com.clone()
    com[:, :, length + count :] = 77.0                # left as it is, as the demand behind the accepted rows
    k[:, :, length + n :] = v[:, :, length + n :] = float("nan")
    new = kernels.dilution_tree_accept(q, k, v, com, length, aux["lse"], path)
    assert new == length + count
    for i in range(b):
        for j in range(h):
            want, rows = ref.accept_f64(q[i, j], k0[i, j], c0[i, j], length, aux["lse"][i, j], path[i])
            seen = torch.cat([k0[i, j, :length], k0[i, j][rows]])
            delta = ref.score_error(q[i, j], seen, d) + 2.0 ** -22 * aux["lse"][i, j].abs().max().item()
            # each bid's relative error (affinity, exp2), and the fp32 sum of the count + 1 terms
            bids = want - torch.cat([c0[i, j, :length].double(), torch.zeros(count, dtype=torch.float64, device=want.device)])
            bound = (2 * delta + 2.0 ** -20) * bids.abs() + (count + 1) * 2.0 ** -24 * want.abs() + 1e-12
            err = (com[i, j, : length + count].double() - want).abs()
            assert bool((err <= bound).all()), (i, j, (err / bound).max().item())
            for cache, old in ((k, k0), (v, v0)):
                assert torch.equal(cache[i, j, :length], old[i, j, :length])
                assert torch.equal(cache[i, j, length : length + count], old[i, j][rows])
                assert torch.equal(cache[i, j, length + count : length + n], old[i, j, length + count : length + n])
                assert bool(torch.isnan(cache[i, j, length + n :]).all())
    assert bool((com[:, :, length + count :] == 77.0).all())


def test_accept_of_wild_device_paths_stays_inside():
    """Entries outside the tree count for nothing and leave their row; the same node twice is taken twice."""
    from dilution import kernels

    length, n, d = 100, 6, 64
    q, k, v, com = _make(21, 1, 2, length, n, d, BF16)
    tree = _tree("chain", n, 0)
    _, aux = kernels.dilution_tree_step(q, k, v, com, length, tree, return_aux=True)
    k0, v0, c0 = k.clone(), v.clone(), com.clone()
    wild = torch.tensor([0, 6, 2, -5], dtype=torch.int32).cuda()
    assert kernels.dilution_tree_accept(q, k, v, com, length, aux["lse"], wild) == length + 4
    for old, cache in ((k0, k), (v0, v)):
        assert torch.equal(cache[:, :, length + 2], old[:, :, length + 2]) and torch.equal(cache[:, :, length], old[:, :, length])
        for r in (1, 3, 4, 5):
            assert torch.equal(cache[:, :, length + r], old[:, :, length + r])
    assert bool((com[:, :, length + 1] == 0).all()) and bool((com[:, :, length + 3] == 0).all())
    for j in range(2):
        want, _ = ref.accept_f64(q[0, j], k0[0, j], c0[0, j], length, aux["lse"][0, j], [0, 2])
        assert (com[0, j, :length] - want[:length]).abs().max().item() < 1e-5
    twice = torch.tensor([1, 1], device="cuda")
    k, v, com = k0.clone(), v0.clone(), c0.clone()
    kernels.dilution_tree_accept(q, k, v, com, length, aux["lse"], twice)
    assert torch.equal(k[:, :, length], k0[:, :, length + 1]) and torch.equal(k[:, :, length + 1], k0[:, :, length + 1])


def test_accept_of_an_absent_node_adds_nothing_to_the_cached_keys():
    from dilution import kernels

    length, n = 64, 3
    q, k, v, com = _make(22, 1, 1, length, n, 64, BF16)
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, [-1, -2, 0], return_aux=True)
    c0 = com.clone()
    kernels.dilution_tree_accept(q, k, v, com, length, aux["lse"], [1])
    assert torch.equal(com[:, :, :length], c0[:, :, :length])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_an_accepted_absent_node_brings_no_nan(dtype):
    """Its query may hold anything: the demand of every position takes the present nodes' bids alone."""
    from dilution import kernels

    length, n, d = 50, 3, 64
    q, k, v, com = _make(25, 1, 2, length, n, d, dtype, strided=False)
    q[:, :, 1] = float("nan")
    _, aux = kernels.dilution_tree_step(q, k, v, com, length, [-1, -2, 0], return_aux=True)
    k0, c0 = k.clone(), com.clone()
    kernels.dilution_tree_accept(q, k, v, com, length, aux["lse"], [0, 1, 2])
    for j in range(2):
        lse = aux["lse"][0, j].clone()
        q2 = q[0, j].clone()
        q2[1] = 0                                     # bids of 0: 2^(0 - inf)
        want, _ = ref.accept_f64(q2, k0[0, j], c0[0, j], length, lse, [0, 1, 2])
        assert (com[0, j, : length + 3].double() - want).abs().max().item() < 1e-5


def test_accept_with_keys_and_values_in_one_buffer():
    """A cache whose values are its keys: the rows move once."""
    from dilution import kernels

    length, n = 70, 8
    q, k, _, com = _make(23, 1, 2, length, n, 64, BF16)
    tree = [-1, 0, 0, 1, 2, 4, 5, 6]
    _, aux = kernels.dilution_tree_step(q, k, k, com, length, tree, return_aux=True)
    k0 = k.clone()
    kernels.dilution_tree_accept(q, k, k, com, length, aux["lse"], [0, 2, 4, 5, 6])
    for r, node in enumerate([0, 2, 4, 5, 6]):
        assert torch.equal(k[:, :, length + r], k0[:, :, length + node])


def test_a_row_without_bids_is_nan_as_its_softmax():
    """Every score of node 1 is -inf: no bids; the others stay."""
    from dilution import kernels

    length, n = 40, 4
    q, k, v, com = _make(24, 1, 1, length, n, 64, F32)
    k[:, :, :, 0] = k[:, :, :, 0].abs() + 0.5
    clean = kernels.dilution_tree_step(q, k, v, com, length, [-1, -1, 0, 1])
    q[:, :, 1] = 0.0
    q[:, :, 1, 0] = -float("inf")
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, [-1, -1, 0, 1], return_aux=True)
    assert bool(torch.isnan(out[:, :, [1, 3]]).all())
    assert torch.equal(out[:, :, [0, 2]], clean[:, :, [0, 2]])


def test_many_slices_and_a_broadcast_query():
    """More slices than one grid takes, and queries that the heads share (a stride of 0)."""
    from dilution import kernels

    b, h, length, n, d = 4400, 15, 3, 2, 16
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(b, 1, n, d, generator=g, device="cuda").to(BF16).expand(b, h, n, d)
    k = torch.randn(b, h, length + n, d, generator=g, device="cuda").to(BF16)
    v = torch.randn(b, h, length + n, d, generator=g, device="cuda").to(BF16)
    com = torch.rand(b, h, length + n, generator=g, device="cuda")
    com[:, :, length:] = 0
    out, aux = kernels.dilution_tree_step(q, k, v, com, length, [-1, 0], return_aux=True)
    for i, j in ((0, 0), (2345, 7), (4369, 1), (4399, 14)):
        one = slice(i, i + 1)
        _check_step(q[one, j : j + 1], k[one, j : j + 1], v[one, j : j + 1], com[one, j : j + 1], length, [[-1, 0]],
                    out[one, j : j + 1], aux["lse"][one, j : j + 1])
    c0 = com.clone()
    kernels.dilution_tree_accept(q, k, v, com, length, aux["lse"], [0, 1])
    for i, j in ((0, 0), (4399, 14)):
        want, _ = ref.accept_f64(q[i, j], k[i, j], c0[i, j], length, aux["lse"][i, j], [0, 1])
        assert (com[i, j].double() - want).abs().max().item() < 1e-5


# ---------------------------------------------------------------------------
# streams, graphs, far offsets


def test_step_and_accept_in_a_graph():
    """One capture serves later trees, paths, queries and demands; every replay equals the eager calls."""
    from dilution import kernels

    b, h, length, n, d = 2, 4, 1100, 10, 64
    q, k, v, com = _make(31, b, h, length, n, d, BF16)
    parents = torch.tensor([_tree("bushy", n, i) for i in range(b)], dtype=torch.int32).cuda()
    path = torch.tensor([[0], [0]], dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c = com.clone()
    with torch.cuda.stream(side):
        out, aux = kernels.dilution_tree_step(q, k, v, c, length, parents, return_aux=True)
        kernels.dilution_tree_accept(q, k, v, c, length, aux["lse"], path)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, aux = kernels.dilution_tree_step(q, k, v, c, length, parents, return_aux=True)
        kernels.dilution_tree_accept(q, k, v, c, length, aux["lse"], path)
    for rep in range(4):
        q2, k2, v2, com2 = _make(40 + rep, b, h, length, n, d, BF16)
        trees = torch.tensor([_tree("bushy", n, 10 * rep + i) for i in range(b)], dtype=torch.int32).cuda()
        for dst, src in ((q, q2), (k, k2), (v, v2), (c, com2), (parents, trees)):
            dst.copy_(src)
        graph.replay()
        want, waux = kernels.dilution_tree_step(q2, k2, v2, com2, length, trees, return_aux=True)
        kernels.dilution_tree_accept(q2, k2, v2, com2, length, waux["lse"], path)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(aux["lse"], waux["lse"]) and torch.equal(c, com2)
        assert torch.equal(k, k2) and torch.equal(v, v2)


def test_two_streams_at_once():
    from dilution import kernels

    states = [_make(50 + i, 2, 8, 3000, 20, 64, BF16) for i in range(2)]
    tree = torch.tensor(_tree("bushy", 20, 4), dtype=torch.int32).cuda()
    want = [kernels.dilution_tree_step(*s, 3000, tree) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [[], []]
    for _ in range(5):
        for i, (st, s) in enumerate(zip(streams, states)):
            with torch.cuda.stream(st):
                got[i].append(kernels.dilution_tree_step(*s, 3000, tree))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


def test_offsets_past_32_bits():
    """Caches of more than 2^31 elements: the last slice's rows, and rows far inside one slice."""
    from dilution import kernels

    for b, h, cap, length, d, n in ((1, 3, 1 << 24, 70, 64, 5), (1, 1, (1 << 25) + 4096, (1 << 25) + 321, 64, 3)):
        g = torch.Generator(device="cuda").manual_seed(1)
        k = torch.zeros(b, h, cap, d, dtype=BF16, device="cuda")
        v = torch.zeros_like(k)
        stop = length + n
        tail = min(stop, 5000)
        k[:, :, stop - tail : stop] = torch.randn(b, h, tail, d, generator=g, device="cuda").to(BF16)
        v[:, :, stop - tail : stop] = torch.randn(b, h, tail, d, generator=g, device="cuda").to(BF16)
        q = (torch.randn(b, h, n, d, generator=g, device="cuda") * 4).to(BF16)
        com = torch.zeros(b, h, cap, device="cuda")
        com[:, :, :length] = 0.5
        parents = _tree("chain", n, 0)
        out, aux = kernels.dilution_tree_step(q, k, v, com, length, parents, return_aux=True)
        j = h - 1
        a = torch.cat([(k[0, j, s : s + (1 << 22)].double() @ q[0, j].double().T) for s in range(0, stop, 1 << 22)])[:stop] / math.sqrt(d)
        a[length:] = a[length:].masked_fill(torch.arange(n, device="cuda")[:, None] > torch.arange(n, device="cuda"), -math.inf)
        p = torch.softmax(a, dim=0)
        base = torch.cat([com[0, j, :length].double(), torch.zeros(n, device="cuda", dtype=torch.float64)])
        demand = base[:, None] + p.cumsum(dim=1)
        share = p / (demand + ref.EPS)
        w = share / (share.sum(0) + ref.EPS)
        want = w[stop - tail :].T @ v[0, j, stop - tail : stop].double()
        spread = w[stop - tail :].T @ v[0, j, stop - tail : stop].double().abs()
        delta = ref.score_error(q[0, j], k[0, j, stop - tail : stop], d) + 2.0 ** -22 * 30
        err = (out[0, j].double() - want).abs()
        assert bool((err <= ref.out_bound(want, spread, BF16, delta)).all()), (cap, err.max().item())
        kernels.dilution_tree_accept(q, k, v, com, length, aux["lse"], list(range(n)))
        got = com[0, j, :stop].double() - base
        assert (got - p.sum(dim=1)).abs().max().item() <= 1e-5
        del k, v, com, a, p, demand, share, w
        torch.cuda.empty_cache()
