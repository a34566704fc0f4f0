"""Decode caches in 4 bits on the GPU: rows written and read back bit for bit, and the decode step
over them against float64 (tests/fp4_reference.py)."""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref
from dilution import kernels
from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]

TYPES = [torch.bfloat16, torch.float16, torch.float32]
WIDTHS = [16, 32, 64, 128, 256]


def _caches(b, h, cap, d, seed=None):
    """K and V caches: cleared, or of rows with any codes and ordinary scales."""
    out = [kernels.alloc_fp4_rows(b, h, cap, d) for _ in range(2)]
    if seed is not None:
        g = torch.Generator(device="cuda").manual_seed(seed)
        for c in out:
            c.codes.copy_(torch.randint(0, 256, c.codes.shape, generator=g, device="cuda", dtype=torch.uint8))
            c.scales.copy_(torch.randint(122, 130, c.scales.shape, generator=g, device="cuda", dtype=torch.uint8))
    return out


def _rows(b, h, t, d, dtype, layout, seed):
    """k and v (b, h, t, d) with channels of different sizes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    scale = torch.exp(torch.randn(h * d, generator=g, device="cuda"))
    if layout == "packed":                                  # views of a (B, T, 3 H D) projection
        qkv = (torch.randn(b, t, 3, h * d, generator=g, device="cuda") * scale).to(dtype).view(b, t, 3 * h * d)
        return [x.view(b, t, h, d).transpose(1, 2) for x in qkv.split(h * d, dim=2)[1:]]
    x = [(torch.randn(b, h, t, d, generator=g, device="cuda") * scale.view(h, 1, d)).to(dtype) for _ in range(2)]
    if layout == "sliced":                                  # every second row of a larger tensor
        return [torch.stack([y, torch.full_like(y, 1e4)], dim=3).flatten(2, 3)[:, :, ::2] for y in x]
    if layout == "odd":                                     # rows that no wide load takes
        return [torch.nn.functional.pad(y, (1, 2))[..., 1 : d + 1] for y in x]
    return x


def _same(cache, codes, scales):
    assert torch.equal(cache.codes.cpu(), codes)
    assert torch.equal(cache.scales.cpu(), scales)


# ---------------------------------------------------------------------------
# rows in and out


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,start,layout", [(1, 0, "packed"), (1, 39, "flat"), (7, 5, "sliced"), (33, 1, "odd"), (300, 17, "packed"),
                                            (513, 0, "flat")])
def test_rows_written_bit_for_bit(d, dtype, t, start, layout):
    b, h, cap = 2, 3, start + t + 1
    kc, vc = _caches(b, h, cap, d, seed=1)
    before = [(c.codes.cpu(), c.scales.cpu()) for c in (kc, vc)]
    k, v = _rows(b, h, t, d, dtype, layout, seed=d + t)
    kernels.dilution_fp4_write(k, v, kc, vc, start)
    for x, cache, (codes, scales) in ((k, kc, before[0]), (v, vc, before[1])):
        codes[:, :, start : start + t], scales[:, :, start : start + t] = ref.quantise(x)
        _same(cache, codes, scales)                         # and no other row
        want = ref.values(codes, scales)[:, :, start : start + t]
        for out in TYPES:
            got = kernels.dilution_fp4_read(kc, vc, start, t, out)[0 if cache is kc else 1]
            assert got.shape == (b, h, t, d) and got.dtype == out and got.is_contiguous()
            assert torch.equal(got.cpu(), want.to(out))


def test_mixed_and_wider_types_are_converted():
    kc, vc = _caches(1, 2, 9, 64)
    k, v = _rows(1, 2, 9, 64, torch.float32, "flat", 3)
    kernels.dilution_fp4_write(k.double(), v.half(), kc, vc, 0)
    _same(kc, *ref.quantise(k))
    _same(vc, *ref.quantise(v.half()))


SPECIALS = [0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.9, 7.0, 7.9]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [16, 64])
def test_ties_extremes_and_what_is_no_number(d, dtype):
    """Ties and their neighbours in every power's block, the type's largest, smallest and subnormal
    values, and blocks with a NaN or an infinity beside ordinary ones."""
    info = torch.finfo(dtype)
    rows = []
    for power in (-8, 0, 9):
        base = torch.tensor(SPECIALS, dtype=torch.float64) * 2.0 ** power
        for x in (base, -base, base * (1 + info.eps), base * (1 - info.eps)):
            rows.append(torch.nn.functional.pad(x, (0, d - len(SPECIALS))))
            rows.append(rows[-1].clamp(max=6.9 * 2.0 ** power))
    step = torch.linspace(-1, 1, d, dtype=torch.float64)
    for top in (info.max, info.max / 1.5, info.tiny, info.tiny * 4, info.smallest_normal * info.eps * 5, info.smallest_normal * 1.9):
        rows.append(step * top)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for at in (0, 5, d - 1):
            x = step.clone()
            x[at] = bad
            rows.append(x)
    rows.append(torch.full((d,), float("nan"), dtype=torch.float64))
    x = torch.stack(rows).to(dtype)[None, None]
    kc, vc = _caches(1, 1, x.shape[2], d)
    kernels.dilution_fp4_write(x.cuda(), -x.cuda(), kc, vc, 0)
    for cache, rows in ((kc, x), (vc, -x)):
        codes, scales = ref.quantise(rows)
        _same(cache, codes, scales)
        for out in TYPES:
            got = kernels.dilution_fp4_read(kc, vc, 0, x.shape[2], out)[0 if cache is kc else 1].cpu()
            torch.testing.assert_close(got, ref.values(codes, scales).to(out), rtol=0, atol=0, equal_nan=True)


def test_a_cleared_cache_and_empty_ranges():
    kc, vc = _caches(2, 2, 5, 32)
    for x in kernels.dilution_fp4_read(kc, vc, 0, 5):
        assert x.shape == (2, 2, 5, 32) and not x.any()
    for x in kernels.dilution_fp4_read(kc, vc, 5, 0):
        assert x.shape == (2, 2, 0, 32)
    empty = torch.zeros(2, 2, 0, 32, device="cuda")
    kernels.dilution_fp4_write(empty, empty, kc, vc, 5)
    assert not kc.codes.any()
    none = [kernels.alloc_fp4_rows(0, 2, 5, 32) for _ in range(2)]
    kernels.dilution_fp4_write(torch.zeros(0, 2, 1, 32, device="cuda"), torch.zeros(0, 2, 1, 32, device="cuda"), *none, 0)
    assert kernels.dilution_fp4_read(*none, 0, 5)[0].shape == (0, 2, 5, 32)
    q = torch.zeros(0, 2, 1, 32, device="cuda")
    assert kernels.dilution_decode_step_fp4(q, *none, torch.zeros(0, 2, 5, device="cuda"), 3).shape == (0, 2, 1, 32)


@pytest.mark.parametrize("start", [0, 3, 9, -2, -4, 12, 13, -(1 << 62), (1 << 63) - 1, -(1 << 63)])
def test_a_device_start_drops_rows_outside(start):
    b, h, cap, t, d = 1, 2, 13, 4, 64
    kc, vc = _caches(b, h, cap, d, seed=2)
    codes, scales = kc.codes.cpu(), kc.scales.cpu()
    k, v = _rows(b, h, t, d, torch.bfloat16, "flat", 4)
    kernels.dilution_fp4_write(k, v, kc, vc, torch.tensor([start], device="cuda"))
    new_codes, new_scales = ref.quantise(k)
    for i in range(t):
        if 0 <= start + i < cap:
            codes[:, :, start + i], scales[:, :, start + i] = new_codes[:, :, i], new_scales[:, :, i]
    _same(kc, codes, scales)


def test_positions_past_four_gigabytes():
    """The last slice of caches whose codes pass 2^32 bytes: rows written, read and stepped over."""
    b, h, cap, d, length = 1, 5, 8_500_000, 256, 700
    kc, vc = _caches(b, h, cap, d)
    k, v = _rows(b, h, length, d, torch.bfloat16, "packed", 5)
    kernels.dilution_fp4_write(k, v, kc, vc, 0)
    tail = _rows(b, h, 3, d, torch.bfloat16, "flat", 6)
    kernels.dilution_fp4_write(*tail, kc, vc, cap - 3)
    for got, want in zip(kernels.dilution_fp4_read(kc, vc, cap - 3, 3, torch.float32), tail):
        assert torch.equal(got.cpu(), ref.values(*ref.quantise(want)).float())
    q = torch.randn(b, h, 1, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))
    com = torch.rand(b, h, cap, device="cuda")
    com[:, :, length - 1] = 0
    small = [kernels.Fp4Rows(c.codes[:, :, :length].contiguous(), c.scales[:, :, :length].contiguous()) for c in (kc, vc)]
    com_small = com[:, :, :length].contiguous()
    out = kernels.dilution_decode_step_fp4(q, kc, vc, com, length)
    assert torch.equal(out, kernels.dilution_decode_step_fp4(q, *small, com_small, length))
    assert torch.equal(com[:, :, :length], com_small)


# ---------------------------------------------------------------------------
# the decode step


def _state(b, h, length, room, d, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cap = length + room
    caches = []
    for _ in range(2):
        codes, scales = ref.quantise(torch.randn(b, h, cap, d, generator=g, device="cuda"))
        caches.append(kernels.Fp4Rows(codes.cuda(), scales.cuda()))
    q = (torch.randn(b, 1, h * d, generator=g, device="cuda") * scale).to(dtype).view(b, 1, h, d).transpose(1, 2)
    com = torch.rand(b, h, cap, generator=g, device="cuda") * 3
    com[:, :, length - 1] = 0
    return q, *caches, com


def _check(q, kc, vc, before, out, com, length):
    kv, vv = ref.values(kc.codes, kc.scales), ref.values(vc.codes, vc.scales)
    for i in range(q.shape[0]):
        for j in range(q.shape[1]):
            want, new, spread, p = ref.step_f64(q[i, j, 0], kv[i, j], vv[i, j], before[i, j], length)
            err = ref.share_error(q[i, j, 0].float(), kv[i, j], length)
            bound = ref.out_bound(want, spread, q.dtype, err, length)
            assert ((out[i, j, 0].double() - want).abs() <= bound).all(), (i, j, ((out[i, j, 0].double() - want).abs() / bound).max())
            # a key's demand: its bid's error, and the sum rounded once
            bound = err * p + 2.0 ** -24 * new[:length]
            assert ((com[i, j, :length].double() - new[:length]).abs() <= bound + 1e-30).all()
    assert torch.equal(com[:, :, length:], before[:, :, length:])


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,h,length,room", [(1, 1, 1, 0), (2, 3, 2, 5), (1, 2, 65, 3), (3, 1, 255, 0), (1, 5, 1000, 24), (2, 1, 5003, 1),
                                             (1, 1, 20011, 2)])
def test_step_against_float64(d, dtype, b, h, length, room):
    q, kc, vc, com = _state(b, h, length, room, d, dtype, seed=length + d)
    before, held = com.clone(), [x.clone() for x in (*kc, *vc)]
    out = kernels.dilution_decode_step_fp4(q, kc, vc, com, length)
    assert out.shape == (b, h, 1, d) and out.dtype == dtype
    _check(q, kc, vc, before, out, com, length)
    assert all(torch.equal(x, y) for x, y in zip((*kc, *vc), held))
    # the same call, the same bits
    again = before.clone()
    assert torch.equal(kernels.dilution_decode_step_fp4(q, kc, vc, again, length), out) and torch.equal(again, com)


@pytest.mark.parametrize("n,length,d", [(170, 300, 64), (200, 2047, 32), (300, 700, 256), (600, 130, 16), (257, 4100, 64)])
def test_many_slices(n, length, d):
    """From 160 slices on one workgroup takes a slice, where its keys fit."""
    q, kc, vc, com = _state(n, 1, length, 1, d, torch.bfloat16, seed=n)
    before = com.clone()
    out = kernels.dilution_decode_step_fp4(q, kc, vc, com, length)
    at = [0, 1, n // 2, n - 1]
    pick = lambda c: kernels.Fp4Rows(c.codes[at], c.scales[at])                                # noqa: E731
    _check(q[at], pick(kc), pick(vc), before[at], out[at], com[at], length)


def test_more_slices_than_a_grid_dimension():
    n, length, d = 70000, 3, 16
    q, kc, vc, com = _state(n, 1, length, 0, d, torch.float32, seed=1)
    before = com.clone()
    out = kernels.dilution_decode_step_fp4(q, kc, vc, com, length)
    at = [0, 65534, 65535, 65536, n - 1]
    pick = lambda c: kernels.Fp4Rows(c.codes[at], c.scales[at])                                # noqa: E731
    _check(q[at], pick(kc), pick(vc), before[at], out[at], com[at], length)
    k, v = kernels.dilution_fp4_read(kc, vc, 0, length, torch.float32)
    other = [kernels.alloc_fp4_rows(n, 1, length, d) for _ in range(2)]
    kernels.dilution_fp4_write(k, v, *other, 0)
    assert torch.equal(kernels.dilution_fp4_read(*other, 0, length, torch.float32)[1], v)


@pytest.mark.parametrize("scale", [0.0, 1e-3, 40.0])
@pytest.mark.parametrize("length", [700, 9000])
def test_flat_and_peaked_rows(scale, length):
    """Equal affinities, and rows whose bids lie on few keys."""
    q, kc, vc, com = _state(2, 2, length, 0, 64, torch.float32, seed=3, scale=scale)
    com[:, 0] = 0                                           # no demand yet: shares of p / (p + eps)
    before = com.clone()
    out = kernels.dilution_decode_step_fp4(q, kc, vc, com, length)
    _check(q, kc, vc, before, out, com, length)


@pytest.mark.parametrize("b,h,length,d", [(1, 2, 1, 64), (1, 2, 2, 16), (2, 3, 257, 128), (1, 3, 9000, 64), (180, 1, 40, 32), (1, 1, 6000, 256)])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_step_that_takes_the_new_rows(b, h, length, d, dtype):
    """With k1 and v1: the bits of a write and a step."""
    q, kc, vc, com = _state(b, h, length, 2, d, dtype, seed=9)
    k1, v1 = _rows(b, h, 1, d, dtype, "packed", 8)
    other = [kernels.Fp4Rows(c.codes.clone(), c.scales.clone()) for c in (kc, vc)]
    com2 = com.clone()
    kernels.dilution_fp4_write(k1, v1, *other, length - 1)
    want = kernels.dilution_decode_step_fp4(q, *other, com2, length)
    out = kernels.dilution_decode_step_fp4(q, kc, vc, com, length, k1, v1)
    assert torch.equal(out, want) and torch.equal(com, com2)
    for a, c in zip(other, (kc, vc)):
        assert torch.equal(a.codes, c.codes) and torch.equal(a.scales, c.scales)


def test_queries_of_other_types():
    q, kc, vc, com = _state(1, 2, 300, 0, 64, torch.float32, seed=4)
    com2 = com.clone()
    out = kernels.dilution_decode_step_fp4(q.double(), kc, vc, com, 300)
    assert out.dtype == torch.float64
    assert torch.equal(out.float(), kernels.dilution_decode_step_fp4(q, kc, vc, com2, 300))


@pytest.mark.parametrize("length", [300, 9000])
def test_what_is_no_number(length):
    """Behind the length nothing counts, NaN included; a NaN block among the cached keys makes its
    slice's row NaN and no other's."""
    q, kc, vc, com = _state(1, 3, length, 4, 64, torch.bfloat16, seed=6)
    for c in (kc, vc):
        c.scales[:, :, length:] = 255
    com[:, :, length:] = float("nan")
    before = com.clone()
    out = kernels.dilution_decode_step_fp4(q, kc, vc, com, length)
    _check(q, kc, vc, before[:, :, :length], out, com[:, :, :length], length)
    kc.scales[0, 1, length // 2, 0] = 255
    vc.scales[0, 2, length - 3, 1] = 255
    com = before.clone()
    got = kernels.dilution_decode_step_fp4(q, kc, vc, com, length)
    assert torch.equal(got[0, 0], out[0, 0])
    assert got[0, 1].isnan().all() and com[0, 1, :length].isnan().all()
    assert torch.equal(got[0, 2, 0, :32], out[0, 2, 0, :32]) and got[0, 2, 0, 32:].isnan().all()
    # every key of the slice
    kc.scales[0, 0] = 255
    assert kernels.dilution_decode_step_fp4(q, kc, vc, before.clone(), length)[0, 0].isnan().all()


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("n", [1, 40, 143, 144, 256, 257, 300, 512])
def test_both_forms_at_their_border(n, d):
    """The longest contexts that one workgroup takes whole (no workspace), and one key more: float64, and
    a device-resident length on either side of the border."""
    from dilution import _hip

    query = _hip.lib().dil_decode_fp4_workspace_bytes
    short, long = 1, 40000
    assert query(n, short, d) == 0 and query(n, long, d) > 0
    while long - short > 1:
        mid = (short + long) // 2
        short, long = (mid, long) if query(n, mid, d) == 0 else (short, mid)
    kc, vc = _caches(n, 1, long, d, seed=n)
    g = torch.Generator(device="cuda").manual_seed(d)
    q = torch.randn(n, 1, 1, d, generator=g, device="cuda").bfloat16() / 2
    com = torch.rand(n, 1, long, generator=g, device="cuda")
    at = sorted({0, n // 2, n - 1})
    pick = lambda c: kernels.Fp4Rows(c.codes[at], c.scales[at])                                # noqa: E731
    for length in (short, long):
        mine, dev = com.clone(), com.clone()
        out = kernels.dilution_decode_step_fp4(q, kc, vc, mine, length)
        _check(q[at], pick(kc), pick(vc), com[at], out[at], mine[at], length)
        got = kernels.decode_step_fp4_device_length(q, kc, vc, dev, torch.tensor([length], device="cuda"), long)
        assert torch.equal(got, out) and torch.equal(dev, mine)


def test_queries_with_small_and_large_elements():
    """Elements over the whole range of their type beside one another, down to subnormal ones: every
    query element counts to fp32's precision of its block's largest."""
    for dtype, spread in ((torch.bfloat16, 12.0), (torch.float16, 5.0), (torch.float32, 12.0)):
        for d in WIDTHS:
            q, kc, vc, com = _state(2, 2, 900, 0, d, torch.float32, seed=d)
            g = torch.Generator(device="cuda").manual_seed(d + 1)
            q = (q * torch.exp2(-spread * torch.rand(q.shape, generator=g, device="cuda") ** 0.5)).to(dtype)
            q[0, 0, 0, 1::2] *= torch.finfo(dtype).tiny
            q[0, 1] = 0
            before = com.clone()
            out = kernels.dilution_decode_step_fp4(q, kc, vc, com, 900)
            _check(q, kc, vc, before, out, com, 900)


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("value", [1.9375, 1.0, 1.99999988079071044921875, 0.03125 + 2.0 ** -20])
def test_the_largest_sums_of_a_block(d, value):
    """Every product of a block as large as can be and of one sign, but one of the smallest code: the
    small one counts (its loss would be 500 times the bound).  Small block powers keep the bids apart."""
    length, b, h = 300, 1, 2
    g = torch.Generator().manual_seed(d)
    sign = torch.randint(0, 2, (d,), generator=g)
    q = (value * (1 - 2 * sign.float())).expand(b, h, 1, d).contiguous().cuda()
    code = (7 + 8 * sign).expand(b, h, length, d).clone()   # 6 times the query's sign
    at = torch.randint(0, d, (b, h, length, 1), generator=g)
    code.scatter_(3, at, 1 + 8 * torch.randint(0, 2, at.shape, generator=g))       # 0.5, either sign
    kc = kernels.Fp4Rows((code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8).cuda(),
                         torch.full((b, h, length, d // min(32, d)), 127 - 9, dtype=torch.uint8, device="cuda"))
    _, _, vc, com = _state(b, h, length, 0, d, torch.float32, seed=1)
    com[:] = 0.5 / length
    before = com.clone()
    out = kernels.dilution_decode_step_fp4(q, kc, vc, com, length)
    _check(q, kc, vc, before, out, com, length)


def test_a_query_that_is_no_number():
    """A NaN or an infinity in a query makes its slice's row NaN and no other's."""
    for length in (300, 9000):
        q, kc, vc, com = _state(2, 2, length, 0, 64, torch.bfloat16, seed=8)
        want = kernels.dilution_decode_step_fp4(q, kc, vc, com.clone(), length)
        for bad in (float("nan"), float("inf"), -float("inf")):
            x, c = q.clone(), com.clone()
            x[0, 1, 0, 40] = bad
            out = kernels.dilution_decode_step_fp4(x, kc, vc, c, length)
            assert out[0, 1].isnan().all() and c[0, 1].isnan().all()
            for i, j in ((0, 0), (1, 0), (1, 1)):
                assert torch.equal(out[i, j], want[i, j])


def test_one_cache_for_both_is_refused():
    q, kc, vc, com = _state(1, 2, 30, 0, 64, torch.bfloat16, seed=2)
    for pair in ((kc, kc), (kc, kernels.Fp4Rows(vc.codes, kc.scales)), (kernels.Fp4Rows(vc.codes, kc.scales), vc)):
        with pytest.raises(ValueError, match="two caches"):
            kernels.dilution_fp4_write(q, q, *pair, 3)
        with pytest.raises(ValueError, match="two caches"):
            kernels.dilution_decode_step_fp4(q, *pair, com, 30, q, q)
    kernels.dilution_decode_step_fp4(q, kc, kc, com, 30)    # reading one for both writes nothing


def test_caches_that_share_bytes_are_refused():
    b, h, cap, d = 1, 2, 32, 64
    rows = b * h * cap
    q = torch.randn(b, h, 1, d, device="cuda")
    buf = torch.zeros(4 * rows * d // 2, dtype=torch.uint8, device="cuda")
    codes = lambda at: buf[at : at + rows * d // 2].view(b, h, cap, d // 2)
    scales = lambda at: buf[at : at + rows * d // 32].view(b, h, cap, d // 32)
    com = torch.zeros(b, h, cap, device="cuda")
    size, end = rows * d // 2, rows * d // 32
    F = kernels.Fp4Rows
    for kc, vc in ((F(codes(0), scales(2 * size)), F(codes(size - 16), scales(3 * size))),          # codes and codes
                   (F(codes(0), scales(2 * size)), F(codes(size), scales(2 * size + end - 8))),      # scales and scales
                   (F(codes(0), scales(size - 8)), F(codes(2 * size), scales(3 * size))),            # one cache's own two
                   (F(codes(0), scales(3 * size - 8)), F(codes(2 * size), scales(3 * size)))):       # scales and the other's codes
        with pytest.raises(ValueError, match="two caches"):
            kernels.dilution_fp4_write(q, q, kc, vc, 3)
        with pytest.raises(ValueError, match="two caches"):
            kernels.dilution_decode_step_fp4(q, kc, vc, com, 20, q, q)
    assert not buf.any() and not com.any()
    # parts of one buffer that only touch are two caches
    kc, vc = F(codes(0), scales(2 * size)), F(codes(size), scales(2 * size + end))
    kernels.dilution_fp4_write(q, q, kc, vc, 3)
    assert torch.equal(kc.codes, vc.codes) and torch.equal(kc.scales, vc.scales) and kc.codes.any()


@pytest.mark.parametrize("b,h,top,d", [(1, 2, 300, 64), (2, 3, 9000, 64), (170, 1, 9000, 32), (1, 1, 9000, 256), (3, 1, 5000, 16)])
@pytest.mark.parametrize("new", [False, True])
def test_a_device_length_gives_the_same_bits(b, h, top, d, new):
    q, kc, vc, com = _state(b, h, top, 3, d, torch.bfloat16, seed=11)
    rows = _rows(b, h, 1, d, torch.bfloat16, "flat", 12) if new else (None, None)
    ws = kernels.decode_fp4_workspace(b, h, top, d, "cuda")
    for length in sorted({1, 2, 63, 256, 300, top // 2, top - 1, top} & set(range(1, top + 1))):
        com[:, :, length - 1] = 0
        host, dev = com.clone(), com.clone()
        held = [kernels.Fp4Rows(c.codes.clone(), c.scales.clone()) for c in (kc, vc)]
        want = kernels.dilution_decode_step_fp4(q, kc, vc, host, length, *rows)
        out = torch.full((b, h, d), float("nan"), dtype=torch.bfloat16, device="cuda")
        got = kernels.decode_step_fp4_device_length(q, *held, dev, torch.tensor([length], device="cuda"), top, *rows, out=out,
                                                    workspace=ws.fill_(255))
        assert got.data_ptr() == out.data_ptr() and torch.equal(got, want) and torch.equal(host, dev), length
        assert all(torch.equal(x, y) for a, c in zip(held, (kc, vc)) for x, y in zip(a, c))


@pytest.mark.parametrize("top", [300, 9000])
def test_device_lengths_outside_are_clamped(top):
    q, kc, vc, com = _state(1, 2, top, 3, 64, torch.bfloat16, seed=13)
    k1, v1 = _rows(1, 2, 1, 64, torch.bfloat16, "flat", 14)
    held, before = [x.clone() for x in (*kc, *vc)], com.clone()
    for none in (0, -5, -(1 << 63)):
        out = kernels.decode_step_fp4_device_length(q, kc, vc, com, torch.tensor([none], device="cuda"), top, k1, v1)
        assert not out.any() and torch.equal(com, before)
        assert all(torch.equal(x, y) for x, y in zip((*kc, *vc), held))
    want = kernels.dilution_decode_step_fp4(q, kc, vc, before, top)
    out = kernels.decode_step_fp4_device_length(q, kc, vc, com, torch.tensor([(1 << 63) - 1], device="cuda"), top)
    assert torch.equal(out, want) and torch.equal(com, before)


def test_device_length_refusals():
    q, kc, vc, com = _state(1, 2, 300, 0, 64, torch.bfloat16, seed=15)
    step, n = kernels.decode_step_fp4_device_length, torch.tensor([5], device="cuda")
    for bad in (n.int(), n.repeat(2), n.cpu()):
        with pytest.raises(ValueError, match="length"):
            step(q, kc, vc, com, bad, 300)
    for out in (torch.empty(1, 2, 64, device="cuda"), torch.empty(1, 2, 32, device="cuda", dtype=q.dtype), torch.empty(1, 2, 64, dtype=q.dtype)):
        with pytest.raises(ValueError, match="out"):
            step(q, kc, vc, com, n, 300, out=out)
    long = _state(1, 2, 9000, 0, 64, torch.bfloat16, seed=15)        # a length that needs a workspace
    good = kernels.decode_fp4_workspace(1, 2, 9000, 64, "cuda")
    for ws in (good[:-1], good.cpu(), good.float(), good.repeat(2)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            step(*long, n, 9000, workspace=ws)
    with pytest.raises(ValueError, match="start"):
        kernels.dilution_fp4_write(q, q, kc, vc, torch.tensor([5], device="cuda", dtype=torch.int32))


def test_two_streams_and_a_second_thread():
    """Calls on two streams at once, and from a thread of their own, give the bits of calls one by one."""
    import threading

    states = [_state(2, 4, 9000, 1, 64, torch.bfloat16, seed=s) for s in (21, 22)]
    want = []
    for q, kc, vc, com in states:
        c = com.clone()
        want.append((kernels.dilution_decode_step_fp4(q, kc, vc, c, 9000), c))
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        q, kc, vc, com = states[i]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            for _ in range(5):
                c = com.clone()
                out = kernels.dilution_decode_step_fp4(q, kc, vc, c, 9000)
            got[i] = (out, c)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for (a, b), (x, y) in zip(got, want):
        assert torch.equal(a, x) and torch.equal(b, y)


@pytest.mark.parametrize("top", [200, 6000])
def test_a_captured_loop_of_steps(top):
    """One graph of a write, a step and the counters: every replay against the eager steps, with
    eager work between; two graphs side by side."""
    b, h, d, first = 2, 3, 64, 5
    g = torch.Generator(device="cuda").manual_seed(31)
    tokens = [torch.randn(3, b, h, 1, d, generator=g, device="cuda").bfloat16() for _ in range(8)]
    loops = []
    for _ in range(2):
        kc, vc = _caches(b, h, top, d)
        com = torch.zeros(b, h, top, device="cuda")
        start = _rows(b, h, first, d, torch.bfloat16, "flat", 32)
        kernels.dilution_fp4_write(*start, kc, vc, 0)
        pos, live = torch.tensor([first], device="cuda"), torch.tensor([first + 1], device="cuda")
        q, k1, v1 = (torch.zeros(b, h, 1, d, dtype=torch.bfloat16, device="cuda") for _ in range(3))
        out, ws = torch.zeros(b, h, d, dtype=torch.bfloat16, device="cuda"), kernels.decode_fp4_workspace(b, h, top, d, "cuda")

        def body(fused, kc=kc, vc=vc, com=com, pos=pos, live=live, q=q, k1=k1, v1=v1, out=out, ws=ws):
            if fused:
                kernels.decode_step_fp4_device_length(q, kc, vc, com, live, top, k1, v1, out=out, workspace=ws)
            else:
                kernels.dilution_fp4_write(k1, v1, kc, vc, pos)
                kernels.decode_step_fp4_device_length(q, kc, vc, com, live, top, out=out, workspace=ws)
            pos.add_(1)
            live.add_(1)

        loops.append((body, kc, vc, com, pos, live, (q, k1, v1), out))
    graphs = []
    side = torch.cuda.Stream()
    for i, loop in enumerate(loops):
        keep = [x.clone() for x in (*loop[1], *loop[2], loop[3], loop[4], loop[5])]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            loop[0](i == 1)                                 # warm-up
        torch.cuda.current_stream().wait_stream(side)
        for x, y in zip((*loop[1], *loop[2], loop[3], loop[4], loop[5]), keep):
            x.copy_(y)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loop[0](i == 1)
        graphs.append(graph)
    ek, ev = _caches(b, h, top, d)
    ecom = torch.zeros(b, h, top, device="cuda")
    kernels.dilution_fp4_write(*_rows(b, h, first, d, torch.bfloat16, "flat", 32), ek, ev, 0)
    for step, token in enumerate(tokens):
        length = first + step + 1
        kernels.dilution_fp4_write(token[1], token[2], ek, ev, length - 1)
        want = kernels.dilution_decode_step_fp4(token[0], ek, ev, ecom, length)
        for loop in loops:
            for x, y in zip(loop[6], token):
                x.copy_(y)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, kc, vc, com, pos, live, _, out in loops:
            assert torch.equal(out.view_as(want), want) and torch.equal(com, ecom), step
            assert torch.equal(kc.codes, ek.codes) and torch.equal(vc.scales, ev.scales) and int(live) == length + 1
