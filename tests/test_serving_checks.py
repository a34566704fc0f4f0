"""What the tree step, the acceptance and the eviction refuse, on the CPU: host
checks of the Python layer and argument errors of the C entry points, all before
any launch (the stand-in addresses are never dereferenced)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from dilution import _hip, cache, kernels
from dilution.lm import DilutionLM, Eviction, LMConfig


def _state(b=2, h=3, cap=40, n=4, d=64, dtype=torch.bfloat16):
    q = torch.zeros(b, h, n, d, dtype=dtype)
    k = torch.zeros(b, h, cap, d, dtype=dtype)
    return q, k, k.clone(), torch.zeros(b, h, cap)


PARENTS = [-1, 0, 1, 1]


def test_tree_step_refusals():
    q, k, v, com = _state()
    step = kernels.dilution_tree_step
    for bad in ([-1, 1, 0, 0], [0, 0, 0, 0], [-1, 0, 1, -3], torch.tensor([[-1, 0, 1, 3]] * 2)):
        with pytest.raises(ValueError, match="parent"):
            step(q, k, v, com, 36, bad)
    with pytest.raises(ValueError, match="parents"):
        step(q, k, v, com, 36, [-1, 0, 1])
    with pytest.raises(ValueError, match="parents"):
        step(q, k, v, com, 36, torch.zeros(3, 4, dtype=torch.int32) - 1)
    with pytest.raises(ValueError, match="int32 or int64"):
        step(q, k, v, com, 36, torch.zeros(4) - 1)
    for length in (37, -1, 1 << 40, (1 << 63) - 1):
        with pytest.raises(ValueError, match="capacity"):
            step(q, k, v, com, length, PARENTS)
    with pytest.raises(ValueError, match="dtype"):
        step(q.float(), k, v, com, 36, PARENTS)
    with pytest.raises(ValueError, match="dtype"):
        step(q.double(), k.double(), v.double(), com, 36, PARENTS)
    with pytest.raises(ValueError, match="1 to 64"):
        step(*_state(n=65, cap=100), 0, [-1] * 65)
    with pytest.raises(ValueError, match="1 to 64"):
        step(q[:, :, :0], k, v, com, 36, torch.zeros(0, dtype=torch.int32))
    with pytest.raises(ValueError, match="match the cache"):
        step(q[:, :2], k, v, com, 36, PARENTS)
    with pytest.raises(ValueError, match="contiguous"):
        step(q, k.transpose(1, 2).contiguous().transpose(1, 2), v, com, 36, PARENTS)
    with pytest.raises(ValueError, match="committed"):
        step(q, k, v, com[:, :, :-1], 36, PARENTS)
    with pytest.raises(ValueError, match="head_dim"):
        step(*_state(d=48), 36, PARENTS)
    with pytest.raises(RuntimeError, match="no CPU path"):
        step(q, k, v, com, 36, PARENTS)


def test_tree_accept_refusals():
    q, k, v, com = _state()
    lse = torch.zeros(2, 3, 4)
    accept = kernels.dilution_tree_accept
    for bad in ([0, 0], [1, 0], [0, 4], [-1], [[0, 1], [2, 1]]):
        with pytest.raises(ValueError, match="path"):
            accept(q, k, v, com, 36, lse, bad)
    with pytest.raises(ValueError, match="path"):
        accept(q, k, v, com, 36, lse, [[0, 1]] * 3)
    with pytest.raises(ValueError, match="lse"):
        accept(q, k, v, com, 36, lse[:, :, :3], [0, 1])
    with pytest.raises(ValueError, match="lse"):
        accept(q, k, v, com, 36, lse.double(), [0, 1])
    with pytest.raises(ValueError, match="capacity"):
        accept(q, k, v, com, 37, lse, [0, 1])
    with pytest.raises(ValueError, match="dtype"):
        accept(q.half(), k, v, com, 36, lse, [0, 1])
    with pytest.raises(RuntimeError, match="no CPU path"):
        accept(q, k, v, com, 36, lse, [0, 1])


def test_evict_refusals():
    _, k, v, com = _state()
    evict = kernels.dilution_evict
    for keep in (0, -1, 41):
        with pytest.raises(ValueError, match="keep"):
            evict(k, v, com, 40, keep)
    for first, recent in ((-1, 0), (0, -1), (6, 5), (11, 0), (0, 11), (1 << 62, 1 << 62)):
        with pytest.raises(ValueError, match="first and recent"):
            evict(k, v, com, 40, 10, first, recent)
    for length in (0, 41):
        with pytest.raises(ValueError, match="length"):
            evict(k, v, com, length, 1)
    with pytest.raises(ValueError, match="dtype"):
        evict(k, v.half(), com, 40, 10)
    with pytest.raises(ValueError, match="both"):
        evict(k, v[:, :, :-1].contiguous(), com, 40, 10)
    with pytest.raises(ValueError, match="contiguous"):
        evict(k, v, com.transpose(0, 1).contiguous().transpose(0, 1), 40, 10)
    with pytest.raises(RuntimeError, match="no CPU path"):
        evict(k, v, com, 40, 10)


def test_cache_and_model_refusals():
    _, k, v, com = _state()
    c = {"k": k, "v": v, "len": 38, "committed": com}
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="capacity"):
        cache.tree_step(q, q, q, c, PARENTS)
    with pytest.raises(ValueError, match="moved on"):
        cache.accept_tree(c, {"q": q, "lse": None, "len": 37}, [0])
    assert cache.evict_cache(c, 38) is c
    for bad in (dict(limit=10, keep=10), dict(limit=100, keep=50, first=30, recent=21), dict(limit=9, keep=5, first=-1),
                dict(limit=9, keep=5, first=0, recent=0)):
        with pytest.raises(ValueError, match="eviction"):
            Eviction(**bad)
    mixed = DilutionLM(LMConfig(vocab_size=32, n_layers=2, d_model=32, n_heads=2, layer_attention=["dilution", "softmax"]))
    idx = torch.zeros(1, 4, dtype=torch.long)
    with pytest.raises(ValueError, match="production"):
        mixed.tree_step(idx, [-1, 0, 1, 2], [])
    with pytest.raises(ValueError, match="production"):
        mixed.generate_drafted(idx, 2, None)
    with pytest.raises(ValueError, match="production"):
        mixed.generate(idx, 2, eviction=Eviction(limit=200, keep=100))
    with pytest.raises(ValueError, match="graph=False"):
        mixed.generate(idx, 2, graph=True, eviction=Eviction(limit=200, keep=100))


@pytest.fixture(scope="module")
def lib():
    return _hip.lib()


def _fake(i):
    return ctypes.c_void_p(4096 * (i + 1))


def _rows(i, heads=3, n=4, d=64):
    return ctypes.byref(_hip.Rows(4096 * (i + 1), heads * n * d, n * d, d))


BIG = 1 << 50


def test_c_tree_step_argument_errors(lib):
    def step(batch=2, heads=3, nodes=4, cap=40, length=36, d=64, dtype=1, stride=0, ws=BIG, q=_rows(0), out=_rows(1),
             ptrs=None):
        p = ptrs or [_fake(i) for i in range(6)]
        return lib.dil_tree_step(q, p[0], p[1], p[2], batch, heads, nodes, cap, length, p[3], stride, d, dtype, out, p[4],
                                 p[5], ws, None)

    assert step(d=48) == -1
    assert step(dtype=3) == -2
    need = lib.dil_tree_workspace_bytes(6, 36, 4, 64, 1)
    assert need > 0 and step(ws=need - 1) == -3
    for bad in (dict(nodes=0), dict(nodes=65, cap=200), dict(length=37), dict(length=-1), dict(batch=0), dict(heads=0),
                dict(stride=-1), dict(cap=1 << 31), dict(length=(1 << 62)), dict(heads=1 << 16),
                dict(q=_rows(0, d=60)), dict(out=_rows(1, d=60)), dict(q=None), dict(out=None)):
        assert step(**bad) == -4, bad
    for i in range(6):
        p = [_fake(j) for j in range(6)]
        p[i] = None
        assert step(ptrs=p) == -4, i
    for i in (0, 1):
        p = [_fake(j) for j in range(6)]
        p[i] = ctypes.c_void_p(4096 + 8)
        assert step(ptrs=p) == -4, i


def test_c_tree_accept_argument_errors(lib):
    def accept(nodes=4, cap=40, length=36, count=2, d=64, dtype=1, stride=0, q=_rows(0), ptrs=None):
        p = ptrs or [_fake(i) for i in range(5)]
        return lib.dil_tree_accept(q, p[0], p[1], p[2], 2, 3, nodes, cap, length, p[3], p[4], stride, count, d, dtype, None)

    assert accept(d=8) == -1
    assert accept(dtype=-1) == -2
    for bad in (dict(count=0), dict(count=5), dict(nodes=65, cap=200), dict(length=37), dict(stride=-2), dict(q=None)):
        assert accept(**bad) == -4, bad
    for i in range(5):
        p = [_fake(j) for j in range(5)]
        p[i] = None
        assert accept(ptrs=p) == -4, i


def test_c_evict_argument_errors(lib):
    def evict(n=6, cap=40, length=40, keep=10, first=2, recent=3, out_cap=12, d=64, dtype=1, ws=BIG, ptrs=None):
        p = ptrs or [_fake(i) for i in range(8)]
        return lib.dil_evict(p[0], p[1], p[2], n, cap, length, keep, first, recent, out_cap, d, dtype, p[3], p[4], p[5],
                             p[6], p[7], ws, None)

    assert evict(d=512) == -1
    assert evict(dtype=9) == -2
    assert evict(ws=lib.dil_evict_workspace_bytes(6, 40, 10) - 1) == -3
    for bad in (dict(n=0), dict(length=0), dict(length=41), dict(keep=0), dict(keep=41), dict(first=-1), dict(recent=-1),
                dict(first=8), dict(first=1 << 62, recent=1 << 62), dict(out_cap=9), dict(cap=1 << 32, length=1 << 31),
                dict(out_cap=1 << 31)):
        assert evict(**bad) == -4, bad
    for i in range(8):
        p = [_fake(j) for j in range(8)]
        p[i] = None
        assert evict(ptrs=p) == -4, i


def test_entry_points_are_bound():
    for name in ("dil_tree_step", "dil_tree_accept", "dil_evict"):
        assert name in _hip.SIGNATURES
    assert kernels.MAX_TREE_NODES == 64
