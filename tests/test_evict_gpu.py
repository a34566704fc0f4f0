"""Eviction by demand on the GPU: whole numbers and moved rows have to be exact."""

from __future__ import annotations

import math

import pytest
import torch

import serving_reference as ref
from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _cache(seed, b, h, cap, d, dtype):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(b, h, cap, d, generator=g).to(dtype).cuda()
    v = torch.randn(b, h, cap, d, generator=g).to(dtype).cuda()
    return k, v, torch.rand(b, h, cap, generator=g).mul(3).cuda()


def _check(k, v, com, length, keep, first, recent, capacity, got):
    ko, vo, co, index = got
    b, h, _, d = k.shape
    out_cap = max(keep if capacity is None else capacity, keep)
    assert ko.shape == vo.shape == (b, h, out_cap, d) and ko.dtype == vo.dtype == k.dtype
    assert co.shape == (b, h, out_cap) and index.shape == (b, h, keep) and index.dtype == torch.int32
    host = com.cpu()
    for i in range(b):
        for j in range(h):
            want = ref.evict_f64(host[i, j], length, keep, first, recent)
            assert index[i, j].tolist() == want, (i, j)
    rows = index.long()
    assert torch.equal(ko[:, :, :keep], k.gather(2, rows[..., None].expand(-1, -1, -1, d)))
    assert torch.equal(vo[:, :, :keep], v.gather(2, rows[..., None].expand(-1, -1, -1, d)))
    assert torch.equal(co[:, :, :keep].view(torch.int32), com.gather(2, rows).view(torch.int32))
    for t in (ko, vo, co):
        assert bool((t[:, :, keep:] == 0).all())


SHAPES = [
    # b, h, cap, length, keep, first, recent, capacity, d, dtype
    (1, 1, 1, 1, 1, 0, 0, None, 64, BF16),
    (1, 2, 5, 2, 1, 0, 0, 3, 16, BF16),
    (1, 2, 5, 2, 1, 1, 0, 3, 16, F16),
    (1, 2, 5, 2, 1, 0, 1, None, 16, F32),
    (2, 3, 64, 63, 40, 4, 8, 41, 64, BF16),
    (2, 2, 1024, 1023, 1022, 0, 0, None, 64, BF16),
    (1, 2, 1025, 1025, 1025, 3, 5, 1100, 32, BF16),
    (1, 2, 2000, 1500, 20, 10, 10, None, 64, F32),
    (1, 3, 4096, 4096, 2048, 4, 256, None, 64, BF16),
    (1, 2, 5000, 4097, 1, 0, 0, 10, 128, F16),
    (3, 5, 7001, 7001, 2999, 3, 501, 3076, 128, F32),
    (1, 2, 9000, 8191, 5000, 0, 100, None, 256, BF16),
    (2, 1, 20000, 16385, 16384, 0, 0, None, 256, F32),
    (1, 2, 70000, 66001, 30007, 5, 1003, 30100, 64, BF16),
    (1, 1, 200003, 200003, 100001, 7, 0, None, 16, BF16),
    (1, 2, 32768, 32768, 9000, 0, 0, None, 16, BF16),          # the most keys of one workgroup, and one more
    (1, 2, 32769, 32769, 9000, 0, 0, None, 16, BF16),
    (1, 1, 1048600, 1048600, 400000, 6, 18, None, 16, BF16),   # 64 full chunks between, of a length that takes fewer
    (1, 1, 1100000, 1100000, 700001, 0, 0, None, 16, BF16),    # chunks of two blocks
    (1, 2, 50000, 50000, 50000, 0, 0, None, 16, BF16),
    (2, 2, 1000, 900, 500, 4, 8, 512, 64, BF16),               # the most rows that the selection moves, and one more
    (2, 2, 1000, 900, 500, 4, 8, 513, 64, BF16),
    (2, 2, 1000, 900, 12, 4, 8, 512, 64, BF16),
    (1, 2, 50000, 50000, 40, 20, 20, None, 16, BF16),
    (16, 16, 3000, 2999, 1000, 4, 100, 1064, 64, BF16),
]


@pytest.mark.parametrize("b,h,cap,length,keep,first,recent,capacity,d,dtype", SHAPES)
def test_evict(b, h, cap, length, keep, first, recent, capacity, d, dtype):
    from dilution import kernels

    k, v, com = _cache(length, b, h, cap, d, dtype)
    com[:, :, length:] = float("nan")                  # not read
    before = [t.clone() for t in (k, v, com)]
    got = kernels.dilution_evict(k, v, com, length, keep, first, recent, capacity)
    _check(k, v, com, length, keep, first, recent, capacity, got)
    for t, s in zip((k, v, com), before):
        assert torch.equal(t.view(torch.uint8), s.view(torch.uint8))


def _fill(kind, n, g):
    x = torch.rand(n, generator=g)
    if kind == "equal":
        return torch.full((n,), 1.25)
    if kind == "zeros":
        return torch.zeros(n)
    if kind == "signed_zeros":
        return torch.where(x > 0.5, torch.tensor(0.0), torch.tensor(-0.0))
    if kind == "few":
        return (x * 4).floor()
    if kind == "tiny":                                 # denormals and the smallest steps apart
        return (x * 2 ** 20).floor() * 2.0 ** -149
    if kind == "close":                                # equal but for the last bits
        return (1.0 + (x * 64).floor() * 2.0 ** -23)
    if kind == "wild":
        y = torch.randn(n, generator=g) * 1e30
        y[x < 0.1] = math.nan
        y[(x > 0.1) & (x < 0.2)] = math.inf
        y[(x > 0.2) & (x < 0.3)] = -math.inf
        y[x > 0.9] = torch.finfo(torch.float32).min
        return y
    return x.sort(descending=kind == "falling").values


KINDS = ["equal", "zeros", "signed_zeros", "few", "tiny", "close", "wild", "falling", "rising"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length,keep,first,recent", [(700, 300, 2, 50), (5001, 1234, 0, 0), (40000, 25000, 4, 600)])
def test_evict_ties_and_extremes(kind, length, keep, first, recent):
    from dilution import kernels

    k, v, com = _cache(3, 1, 2, length, 16, BF16)
    g = torch.Generator().manual_seed(KINDS.index(kind))
    for j in range(2):
        com[0, j] = _fill(kind, length, g).cuda()
    got = kernels.dilution_evict(k, v, com, length, keep, first, recent)
    _check(k, v, com, length, keep, first, recent, None, got)


def test_evict_moves_every_bit():
    """Rows of NaN payloads and infinities move as they are."""
    from dilution import kernels

    k, v, com = _cache(4, 1, 2, 500, 64, BF16)
    bits = torch.randint(-32768, 32767, k.shape, dtype=torch.int16).cuda()
    k = bits.view(BF16)
    ko, _, _, index = kernels.dilution_evict(k, v, com, 500, 200)
    want = bits.gather(2, index.long()[..., None].expand(-1, -1, -1, 64))
    assert torch.equal(ko.view(torch.int16), want)


def test_evict_of_many_slices():
    """More slices than one grid's y takes."""
    from dilution import kernels

    k, v, com = _cache(9, 4400, 15, 6, 16, BF16)
    got = kernels.dilution_evict(k, v, com, 6, 3, 1, 1, 4)
    sel = [0, 2345, 4369, 4399]
    _check(k[sel], v[sel], com[sel], 6, 3, 1, 1, 4, [t[sel] for t in got])


def test_evict_empty_batch():
    from dilution import kernels

    k, v, com = _cache(5, 1, 2, 50, 64, BF16)
    got = kernels.dilution_evict(k[:0], v[:0], com[:0], 50, 20)
    assert got[0].shape == (0, 2, 20, 64) and got[3].shape == (0, 2, 20)


def test_evict_in_a_graph_and_on_other_streams():
    from dilution import kernels

    shape = (2, 4, 6000, 64, BF16)
    k, v, com = _cache(6, *shape)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.dilution_evict(k, v, com, 5990, 2000, 4, 100, 2500)
    torch.cuda.current_stream().wait_stream(side)
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.dilution_evict(k, v, com, 5990, 2000, 4, 100, 2500)
    with torch.cuda.graph(graph2, pool=graph.pool()):
        got2 = kernels.dilution_evict(k, v, com, 5000, 100)
    for rep in range(4):
        k2, v2, com2 = _cache(60 + rep, *shape)
        for dst, src in ((k, k2), (v, v2), (com, com2)):
            dst.copy_(src)
        for gr, g_out, args in ((graph, got, (5990, 2000, 4, 100, 2500)), (graph2, got2, (5000, 100))):
            gr.replay()
            want = kernels.dilution_evict(k2, v2, com2, *args)
            torch.cuda.synchronize()
            for a, b in zip(g_out, want):
                assert torch.equal(a, b)


def test_evict_offsets_past_32_bits():
    from dilution import kernels

    cap, length, d = 1 << 24, 3000, 64
    k = torch.zeros(1, 3, cap, d, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    com = torch.zeros(1, 3, cap, device="cuda")
    ks, vs, cs = _cache(8, 1, 3, length, d, BF16)
    k[:, :, :length], v[:, :, :length], com[:, :, :length] = ks, vs, cs
    got = kernels.dilution_evict(k, v, com, length, 1000, 4, 10)
    want = kernels.dilution_evict(ks, vs, cs, length, 1000, 4, 10)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del k, v, com, got
    torch.cuda.empty_cache()
    # far rows of one slice, and an output of more than 2^31 elements
    length, keep = (1 << 25) + 777, (1 << 25) + 3
    k = torch.zeros(1, 1, length, d, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    com = torch.rand(1, 1, length, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) + 1.0
    drop = torch.randperm(length - 10, generator=torch.Generator().manual_seed(3))[: length - keep].cuda()
    com[0, 0, drop] = 0.5
    k[0, 0, -5000:] = torch.randn(5000, d, device="cuda").to(BF16)
    ko, vo, co, index = kernels.dilution_evict(k, v, com, length, keep)
    stay = torch.ones(length, dtype=torch.bool, device="cuda")
    stay[drop] = False
    rows = stay.nonzero()[:, 0]
    assert torch.equal(index[0, 0].long(), rows)
    assert torch.equal(ko[0, 0, -4000:], k[0, 0, rows[-4000:]]) and torch.equal(co[0, 0], com[0, 0, rows])
