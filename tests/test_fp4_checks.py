"""What the 4-bit cache's operators refuse, on the CPU: host checks of the Python layer and
argument errors of the C entry points, all before any launch (the stand-in addresses are never
dereferenced); and the test reference's own pins."""

from __future__ import annotations

import ctypes

import pytest
import torch

import fp4_reference as ref
from dilution import _hip, cache, kernels
from dilution.lm import DilutionLM, Eviction, GraphDecoder, LMConfig


def _rows(b=2, h=3, cap=40, d=64):
    return tuple(kernels.alloc_fp4_rows(b, h, cap, d, device="cpu") for _ in range(2))


def test_rows_describe_themselves():
    for d, scales in ((16, 1), (32, 1), (64, 2), (128, 4), (256, 8)):
        k, _ = _rows(d=d)
        assert k.shape == (2, 3, 40, d) and k.device.type == "cpu"
        assert k.codes.shape[3] == d // 2 and k.scales.shape[3] == scales
    for d in (8, 48, 512):
        with pytest.raises(ValueError, match="head_dim"):
            kernels.alloc_fp4_rows(1, 1, 4, d, device="cpu")


def test_write_refusals():
    kc, vc = _rows()
    k = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    write = kernels.dilution_fp4_write
    for start in (37, -1, 1 << 40, (1 << 63) - 1):
        with pytest.raises(ValueError, match="capacity"):
            write(k, k, kc, vc, start)
    with pytest.raises(ValueError, match="capacity"):
        write(torch.zeros(2, 3, 41, 64), torch.zeros(2, 3, 41, 64), kc, vc, 0)
    for bad in (k[:1], k[:, :2], k[..., :32], k[0]):
        with pytest.raises(ValueError, match="match the cache"):
            write(bad, bad, kc, vc, 0)
    with pytest.raises(ValueError, match="match the cache"):
        write(k, k[:, :, :3], kc, vc, 0)
    with pytest.raises(ValueError, match="float"):
        write(k.int(), k.int(), kc, vc, 0)
    for start in (1.0, 2.5, "3", None, [4]):
        with pytest.raises(TypeError):
            write(k, k, kc, vc, start)
    with pytest.raises(RuntimeError, match="no CPU path"):
        write(k, k, kc, vc, 0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        write(k, k, kc, vc, torch.tensor(3))


def _bad_caches():
    kc, vc = _rows()
    F = kernels.Fp4Rows
    yield "both", kc, _rows(cap=41)[0]
    yield "both", kc, _rows(d=128)[0]
    yield "scales", F(kc.codes, kc.scales[..., :1].contiguous()), vc
    yield "scales", kc, F(vc.codes, vc.scales[:, :, :39].contiguous())
    yield "scales", kc, F(vc.codes, vc.scales[0])
    yield "uint8", F(kc.codes.int(), kc.scales), vc
    yield "uint8", kc, F(vc.codes, vc.scales.float())
    yield "contiguous", F(kc.codes.transpose(1, 2).contiguous().transpose(1, 2), kc.scales), vc
    yield "contiguous", kc, F(vc.codes, vc.scales.transpose(0, 1).contiguous().transpose(0, 1))
    yield "head_dim", F(torch.zeros(2, 3, 40, 24, dtype=torch.uint8), kc.scales), F(torch.zeros(2, 3, 40, 24, dtype=torch.uint8), kc.scales)
    yield "aligned", F(torch.zeros(2 * 3 * 40 * 32 + 8, dtype=torch.uint8)[8:].view(2, 3, 40, 32), kc.scales), vc
    yield "aligned", kc, F(vc.codes, torch.zeros(2 * 3 * 40 * 2 + 2, dtype=torch.uint8)[2:].view(2, 3, 40, 2))


@pytest.mark.parametrize("case", range(12))
def test_caches_that_no_operator_takes(case):
    match, kc, vc = list(_bad_caches())[case]
    k = torch.zeros(2, 3, 1, 64)
    with pytest.raises(ValueError, match=match):
        kernels.dilution_fp4_write(k, k, kc, vc, 0)
    with pytest.raises(ValueError, match=match):
        kernels.dilution_fp4_read(kc, vc, 0, 1)
    with pytest.raises(ValueError, match=match):
        kernels.dilution_decode_step_fp4(k, kc, vc, torch.zeros(2, 3, 40), 5)


def test_read_refusals():
    kc, vc = _rows()
    for start, count in ((-1, 2), (0, 41), (39, 2), (0, -1), (1 << 62, 1 << 62), (1, (1 << 63) - 1)):
        with pytest.raises(ValueError, match="capacity"):
            kernels.dilution_fp4_read(kc, vc, start, count)
    for bad in (torch.float64, torch.uint8, torch.int32):
        with pytest.raises(ValueError, match="dtype"):
            kernels.dilution_fp4_read(kc, vc, 0, 1, bad)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.dilution_fp4_read(kc, vc, 0, 1)


def test_step_refusals():
    kc, vc = _rows()
    q, com = torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16), torch.zeros(2, 3, 40)
    step = kernels.dilution_decode_step_fp4
    for length in (0, 41, -1, 1 << 40):
        with pytest.raises(ValueError, match="capacity"):
            step(q, kc, vc, com, length)
    for bad in (q[:1], q[..., :32], torch.zeros(2, 3, 2, 64), q[0]):
        with pytest.raises(ValueError, match="q1"):
            step(bad, kc, vc, com, 5)
    with pytest.raises(ValueError, match="float"):
        step(q.int(), kc, vc, com, 5)
    for bad in (com[:, :, :39], com[0], com[:1]):
        with pytest.raises(ValueError, match="committed"):
            step(q, kc, vc, bad, 5)
    for bad in (com.double(), com.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(ValueError, match="committed"):
            step(q, kc, vc, bad, 5)
    with pytest.raises(ValueError, match="together"):
        step(q, kc, vc, com, 5, k1=q)
    with pytest.raises(ValueError, match="together"):
        step(q, kc, vc, com, 5, v1=q)
    with pytest.raises(ValueError, match="k1"):
        step(q, kc, vc, com, 5, q[:1], q)
    with pytest.raises(ValueError, match="v1"):
        step(q, kc, vc, com, 5, q, q[..., :32])
    with pytest.raises(ValueError, match="dtype"):
        step(q, kc, vc, com, 5, q, q.float())
    for length in (5.0, "5", None):
        with pytest.raises(TypeError):
            step(q, kc, vc, com, length)
    with pytest.raises(RuntimeError, match="no CPU path"):
        step(q, kc, vc, com, 5, q, q)
    with pytest.raises(ValueError, match="length"):
        kernels.decode_step_fp4_device_length(q, kc, vc, com, 5, 40)
    with pytest.raises(ValueError, match="capacity"):
        kernels.decode_step_fp4_device_length(q, kc, vc, com, torch.tensor([5]), 41)


def test_c_entry_argument_errors():
    lib = _hip.lib()
    at = [ctypes.c_void_p(4096 * (i + 1)) for i in range(12)]
    c = _hip.Fp4Cache(4096, 8192)
    off, none = _hip.Fp4Cache(4096 + 8, 8192), _hip.Fp4Cache(0, 8192)
    odd = _hip.Fp4Cache(4096, 8192 + 4)
    rows = _hip.Rows(4096, 3 * 40 * 64, 40 * 64, 64)

    def write(k=rows, b=2, h=3, t=4, start=0, dev=None, cap=40, d=64, dt=1, kc=c, vc=c):
        return lib.dil_fp4_write(ctypes.byref(k), ctypes.byref(rows), b, h, t, start, dev, cap, d, dt, ctypes.byref(kc),
                                 ctypes.byref(vc), None)

    assert write(d=48) == -1 and write(dt=3) == -2
    for bad in (dict(t=0), dict(t=41), dict(start=37), dict(start=-1), dict(b=0), dict(h=1 << 16), dict(cap=1 << 31),
                dict(kc=off), dict(vc=odd), dict(kc=none), dict(k=_hip.Rows(4096, 64, 64, 8)), dict(k=_hip.Rows(4100, 64, 64, 64)),
                dict(k=_hip.Rows(0, 64, 64, 64)), dict(t=(1 << 31) - 1, cap=(1 << 31) - 1)):
        assert write(**bad) == -4, bad

    def read(n=6, cap=40, start=0, t=4, d=64, dt=1, kc=c, k=at[0], v=at[1]):
        return lib.dil_fp4_read(ctypes.byref(kc), ctypes.byref(c), n, cap, start, t, d, dt, k, v, None)

    assert read(d=0) == -1 and read(dt=-1) == -2
    for bad in (dict(n=0), dict(n=1 << 31), dict(t=0), dict(start=-1), dict(start=37), dict(k=None), dict(v=ctypes.c_void_p(4104)),
                dict(kc=off), dict(kc=none)):
        assert read(**bad) == -4, bad

    need = lib.dil_decode_fp4_workspace_bytes(6, 40000, 64)
    assert need > 0 and lib.dil_decode_fp4_workspace_bytes(6, 40, 64) == 0

    def step(q=at[0], k1=None, v1=None, kc=c, vc=c, com=at[1], out=at[2], n=6, cap=40000, length=40000, d=64, dt=1,
             ws=at[3], size=need):
        return lib.dil_decode_step_fp4(q, k1, v1, ctypes.byref(kc), ctypes.byref(vc), com, out, n, cap, length, None, d, dt, ws,
                                       size, None)

    assert step(d=20) == -1 and step(dt=7) == -2 and step(size=need - 1) == -3
    for bad in (dict(q=None), dict(k1=at[4]), dict(v1=at[4]), dict(k1=ctypes.c_void_p(4104), v1=at[4]), dict(kc=off), dict(vc=odd),
                dict(com=None), dict(out=None), dict(n=0), dict(length=0), dict(length=40001), dict(cap=1 << 31, length=4),
                dict(ws=None), dict(q=ctypes.c_void_p(4098))):
        assert step(**bad) == -4, bad
    for n, length in ((0, 5), (-1, 5), (3, 0), (3, -2)):
        assert lib.dil_decode_fp4_workspace_bytes(n, length, 64) == 0
    # a workspace for more keys runs fewer
    for n in (1, 7, 130, 300):
        sizes = [lib.dil_decode_fp4_workspace_bytes(n, x, 64) for x in range(1, 30000, 97)]
        assert sizes == sorted(sizes)


def _packed(length=30, cap=40):
    k, v = _rows(cap=cap)
    return {"k": k, "v": v, "len": length, "committed": torch.zeros(2, 3, cap)}


def test_what_needs_ordinary_rows_says_so():
    c = _packed()
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="unpack_cache"):
        cache.tree_step(q, q, q, c, [-1, 0, 1, 2])
    for keep in (10, 40):
        with pytest.raises(ValueError, match="unpack_cache"):
            cache.evict_cache(c, keep)
    with pytest.raises(ValueError, match="unpack_cache"):
        cache.pack_cache(c)
    with pytest.raises(ValueError, match="4 bits"):
        cache.unpack_cache({"k": q, "v": q, "len": 4, "committed": torch.zeros(2, 3, 4)})
    with pytest.raises(ValueError, match="production"):
        cache.step_cache(q[:, :, :1], q[:, :, :1], q[:, :, :1], c, bid="relu", share_cumsum=True, shift=1.0)
    full = _packed(length=40)
    for step in (lambda: cache.step_cache(q[:, :, :1], q[:, :, :1], q[:, :, :1], full),
                 lambda: cache.append_kv(full, q[:, :, :1], q[:, :, :1])):
        with pytest.raises(ValueError, match="capacity"):
            step()
    assert full["len"] == 40
    with pytest.raises(ValueError, match="bits"):
        cache.begin_cache(q, q, q, bits=8)
    with pytest.raises(ValueError, match="production"):
        cache.begin_cache(q, q, q, bits=4, bid="relu", share_cumsum=True, shift=1.0)


def test_model_refusals():
    cfg = dict(vocab_size=32, n_layers=2, d_model=64, n_heads=4)
    idx = torch.zeros(1, 4, dtype=torch.long)
    model = DilutionLM(LMConfig(**cfg))
    with pytest.raises(ValueError, match="cache_bits"):
        model.generate(idx, 4, cache_bits=4, eviction=Eviction(limit=10, keep=8))
    for other in (dict(attention="softmax"), dict(bid="relu"), dict(layer_attention=["dilution", "softmax"])):
        with pytest.raises(ValueError, match="production"):
            DilutionLM(LMConfig(**cfg, **other)).generate(idx, 4, cache_bits=4)
    with pytest.raises(ValueError, match="4 bits"):
        DilutionLM(LMConfig(**cfg, attention="softmax")).prefill(idx, cache_bits=4)
    mixed = [_packed(), {"k": torch.zeros(2, 3, 40, 64), "v": None, "len": 30, "committed": None}]
    with pytest.raises(ValueError, match="all"):
        GraphDecoder(model, mixed, torch.zeros(2, 1, dtype=torch.long))


# ---------------------------------------------------------------------------
# the reference form, by hand


def test_reference_by_hand():
    x = torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, 6.9, 0.26, 5.01, -0.0, 0.3, 1.0])
    codes, scales = ref.quantise(x)
    assert scales.tolist() == [127]
    want = [0, 0, 1, 1, 2, 2, 4, 4, 0, -1, 6, 0.5, 6, 0, 0.5, 1]
    assert ref.values(codes, scales).tolist() == want
    # 7 rounds beyond 6: the next power
    codes, scales = ref.quantise(torch.cat([torch.tensor([7.0]), x[1:]]))
    assert scales.tolist() == [128] and ref.values(codes, scales)[0] == 8
    for bad in (float("nan"), float("inf"), -float("inf")):
        codes, scales = ref.quantise(torch.cat([x, torch.tensor([bad]), x, x])[:32].view(1, 32))
        assert scales.tolist() == [[255]] and not codes.any() and ref.values(codes, scales).isnan().all()
    codes, scales = ref.quantise(torch.zeros(64))
    assert scales.tolist() == [2, 2] and not ref.values(codes, scales).any()
    assert not ref.values(torch.zeros(1, 32, dtype=torch.uint8), torch.zeros(1, 2, dtype=torch.uint8)).any()


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("scale", [1.0, 1e-30, 3e38, 2.0 ** -130])
def test_reference_errors_are_half_a_step(d, scale):
    """Half a step of a code is at most 1/4 below 2, 1/2 below 4 and 1 above, times the block's power."""
    x = torch.randn(50, d, generator=torch.Generator().manual_seed(d)).clamp(-1, 1) * scale
    codes, scales = ref.quantise(x)
    y = ref.values(codes, scales)
    power = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127).repeat_interleave(min(32, d), dim=1)
    r = x.double().abs() / power
    half = torch.where(r < 2, 0.25, torch.where(r < 4, 0.5, torch.where(r < 7, 1.0, 2.0)))
    assert ((x.double() - y).abs() <= half * power).all()
    assert scale > 1e38 or (r < 7).all()
