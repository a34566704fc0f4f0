"""4-bit decode caches as they are used together: a prompt prefilled and quantised, steps behind it,
read back for the operators that take ordinary rows, and a model that generates on them."""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref
from dilution import cache, kernels
from dilution.lm import DilutionLM, GraphDecoder, LMConfig
from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]


def _rows(b, h, t, d, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(b, t, h, d, generator=g, device="cuda").to(dtype).transpose(1, 2) for _ in range(3)]


@pytest.mark.parametrize("dtype,d,chunk", [(torch.bfloat16, 64, None), (torch.bfloat16, 64, 96), (torch.float16, 32, None), (torch.float32, 128, 64)])
def test_a_prompt_and_steps_behind_it(dtype, d, chunk):
    """The prompt's rows and demand are those of an ordinary cache; each step's output is that of the
    operator on the values held, in float64."""
    b, h, t, room = 2, 3, 210, 12
    q, k, v = _rows(b, h, t, d, dtype, 1)
    y0, plain = cache.begin_cache(q, k, v, capacity=t + room, chunk=chunk)
    y, c = cache.begin_cache(q, k, v, capacity=t + room, chunk=chunk, bits=4)
    assert torch.equal(y, y0) and c["len"] == t and cache.is_packed(c) and c["k"].shape == (b, h, t + room, d)
    assert torch.equal(c["committed"], plain["committed"])
    packed = cache.pack_cache(plain)
    for one in ("k", "v"):
        assert all(torch.equal(x, z) for x, z in zip(packed[one], c[one]))
    codes, scales = ref.quantise(k)
    assert torch.equal(c["k"].codes[:, :, :t].cpu(), codes) and torch.equal(c["k"].scales[:, :, :t].cpu(), scales)
    for i in range(room):
        q1, k1, v1 = _rows(b, h, 1, d, dtype, 10 + i)
        before = c["committed"].clone()
        if i % 3 == 2:                                      # appended apart
            length = cache.append_kv(c, k1, v1)
            out = kernels.dilution_decode_step_fp4(q1, c["k"], c["v"], c["committed"], length)
        else:
            out = cache.step_cache(q1, k1, v1, c)
        length = t + i + 1
        assert c["len"] == length and out.dtype == dtype
        kv, vv = ref.values(*c["k"]), ref.values(*c["v"])
        assert torch.equal(kv[:, :, length - 1].cpu(), ref.values(*ref.quantise(k1))[:, :, 0])
        for n in range(b):
            for j in range(h):
                want, new, spread, p = ref.step_f64(q1[n, j, 0], kv[n, j], vv[n, j], before[n, j], length)
                err = ref.share_error(q1[n, j, 0].float(), kv[n, j], length)
                assert ((out[n, j, 0].double() - want).abs() <= ref.out_bound(want, spread, dtype, err, length)).all()
                assert ((c["committed"][n, j].double() - new).abs() <= 1e-30 + 2.0 ** -24 * new + err * torch.nn.functional.pad(p, (0, room - i - 1))).all()
    with pytest.raises(ValueError, match="capacity"):
        cache.step_cache(q1, k1, v1, c)


def test_a_cache_read_back_takes_the_other_operators():
    """Unpacked, a cache takes a tree step and an eviction; its values are the packed cache's, and packing
    it again changes nothing (every value is one of its block's codes)."""
    b, h, t, d = 2, 4, 300, 64
    q, k, v = _rows(b, h, t, d, torch.bfloat16, 3)
    _, c = cache.begin_cache(q, k, v, capacity=t + 8, bits=4)
    plain = cache.unpack_cache(c, capacity=t + 20)
    assert plain["k"].shape == (b, h, t + 20, d) and plain["len"] == t and not plain["k"][:, :, t:].any()
    assert torch.equal(plain["k"].double()[:, :, :t], ref.values(*c["k"])[:, :, :t])
    assert torch.equal(plain["committed"][:, :, :t], c["committed"][:, :, :t]) and not plain["committed"][:, :, t:].any()
    again = cache.unpack_cache(cache.pack_cache(plain, t + 8))
    for one in ("k", "v", "committed"):
        assert torch.equal(again[one], plain[one][:, :, : t + 8])
    q1, k1, v1 = _rows(b, h, 1, d, torch.bfloat16, 4)
    # the ordinary step over the values read back, with the new row's value as it is held
    held1 = ref.values(*ref.quantise(k1)).cuda().bfloat16(), ref.values(*ref.quantise(v1)).cuda().bfloat16()
    out, want = cache.step_cache(q1, k1, v1, c), cache.step_cache(q1, *held1, plain)
    # the two agree but for the order of fp32 sums, and a step of the outputs' rounding
    assert ((out.double() - want.double()).abs() <= 2.0 ** -8 * want.double().abs() + 1e-4).all()
    assert (c["committed"] - plain["committed"][:, :, : t + 8]).abs().max() <= 1e-6
    y, draft = cache.tree_step(*_rows(b, h, 4, d, torch.bfloat16, 5), plain, [-1, 0, 0, 1])
    assert cache.accept_tree(plain, draft, [0, 1]) == t + 3
    small = cache.pack_cache(cache.evict_cache(plain, 64, first=4, recent=16), 80)
    assert small["len"] == 64 and small["k"].shape == (b, h, 80, d)
    cache.step_cache(q1, k1, v1, small)
    assert small["len"] == 65


def _model(seed=0, **kw):
    torch.manual_seed(seed)
    model = DilutionLM(LMConfig(**{**dict(vocab_size=128, n_layers=3, d_model=256, n_heads=4, prefill_chunk=32), **kw}))
    return model.to("cuda", torch.bfloat16).eval()


@pytest.mark.parametrize("heads", [4, 16])
def test_a_model_decodes_on_packed_caches(heads):
    """The fused step, the module-by-module one and the graph's steps: the same step up to the order
    of the projections' sums, and each layer's cache is what its own rows quantise to."""
    model = _model(n_heads=heads)
    idx = torch.randint(0, 128, (2, 50), generator=torch.Generator().manual_seed(5)).cuda()
    _, fused = model.prefill(idx, capacity=60, cache_bits=4)
    _, plain = model.prefill(idx, capacity=60, cache_bits=4)
    _, wide = model.prefill(idx, capacity=60)
    assert all(cache.is_packed(c) for c in fused) and not cache.is_packed(wide[0])
    # layer 0 sees the same rows whatever its cache holds
    held = cache.unpack_cache(fused[0])
    assert torch.equal(held["k"][:, :, :50].double().cpu(), ref.values(*ref.quantise(wide[0]["k"][:, :, :50])))
    token = idx[:, -1:]
    for step in range(6):
        a, b = model.decode_step(token, fused), model.decode_step(token, plain, fused=False)
        # bf16 activations of size 1 through 3 layers of 7 rounded products each
        assert (a - b).abs().max() <= 21 * 2.0 ** -8 * max(1.0, b.abs().max().item())
        assert all(c["len"] == 51 + step for c in fused + plain)
        token = a[:, -1].argmax(dim=-1, keepdim=True)


@pytest.mark.parametrize("fused", [True, False])
def test_graph_steps_match_eager_steps(fused):
    model = _model(1)
    idx = torch.randint(0, 128, (2, 40), generator=torch.Generator().manual_seed(6)).cuda()
    _, eager = model.prefill(idx, capacity=52, cache_bits=4)
    _, graph = model.prefill(idx, capacity=52, cache_bits=4)
    token = idx[:, -1:]
    dec = GraphDecoder(model, graph, token, fused=fused)
    for step in range(12):
        logits = model.decode_step(token, eager, fused=fused)
        token = logits[:, -1].float().argmax(dim=-1, keepdim=True)
        got = dec.step()
        torch.cuda.synchronize()
        assert torch.equal(dec.logits, logits) and torch.equal(got, token), step
        for a, b in zip(eager, graph):
            assert a["len"] == b["len"] == 41 + step and torch.equal(a["committed"], b["committed"])
            assert torch.equal(a["k"].codes, b["k"].codes) and torch.equal(a["v"].scales, b["v"].scales)
    with pytest.raises(ValueError, match="capacity"):
        dec.step()


def test_generation_on_packed_caches():
    model = _model(2)
    idx = torch.randint(0, 128, (3, 30), generator=torch.Generator().manual_seed(7)).cuda()
    a = model.generate(idx, 12, cache_bits=4)
    assert a.shape == (3, 42) and torch.equal(a[:, :30], idx)
    assert torch.equal(a, model.generate(idx, 12, cache_bits=4, graph=True))
    sample = [model.generate(idx, 6, temperature=0.8, cache_bits=4, generator=torch.Generator(device="cuda").manual_seed(1)) for _ in range(2)]
    assert torch.equal(*sample)
    # a batch that the fused projections do not take
    wide = idx[:1].expand(9, -1).contiguous()
    assert model.generate(wide, 5, cache_bits=4).shape == (9, 35)


def test_a_packed_cache_takes_a_quarter():
    model = _model(3)
    idx = torch.randint(0, 128, (2, 64)).cuda()
    size = lambda caches: sum(x.numel() * x.element_size() for c in caches for one in ("k", "v")      # noqa: E731
                              for x in (c[one] if cache.is_packed(c) else [c[one]]))
    packed, plain = model.prefill(idx, 2048, cache_bits=4)[1], model.prefill(idx, 2048)[1]
    assert size(packed) * 64 * 2 == size(plain) * 34
