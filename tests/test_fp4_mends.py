"""Calls on 4-bit caches that are refused before they write, and calls beside them that are taken, on the CPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from dilution import _hip, cache, kernels
from dilution.lm import Block, DilutionLM, LMConfig, SoftmaxAttention


@pytest.mark.parametrize("off", [1, 2, 4, 8, 12])
def test_a_workspace_off_its_alignment_is_refused(off):
    lib = _hip.lib()
    c = _hip.Fp4Cache(4096, 8192)
    need = lib.dil_decode_fp4_workspace_bytes(6, 40000, 64)
    assert need > 0
    at = ctypes.c_void_p
    # refused before any launch: the addresses are never used
    assert lib.dil_decode_step_fp4(at(4096), None, None, ctypes.byref(c), ctypes.byref(c), at(8192), at(12288), 6, 40000, 40000,
                                   None, 64, 1, at(16384 + off), need, None) == -4


@pytest.mark.parametrize("rows", [0, 2, 3])
def test_one_position_is_appended(rows):
    """Not two, of which the second would lie behind the new length, and not none."""
    k, v = (kernels.alloc_fp4_rows(1, 2, 8, 64, device="cpu") for _ in range(2))
    c = {"k": k, "v": v, "len": 5, "committed": torch.zeros(1, 2, 8)}
    x = torch.ones(1, 2, rows, 64)
    with pytest.raises(ValueError, match="one new position"):
        cache.append_kv(c, x, x)
    assert c["len"] == 5 and not k.codes.any()


def test_modules_of_a_callers_own_need_not_know_of_bits():
    """Attention, blocks and models whose begin_cache and prefill take a capacity alone run as they did."""

    class Attention(SoftmaxAttention):
        def begin_cache(self, x, capacity=None):
            return super().begin_cache(x, capacity)

    class Layer(Block):
        def begin_cache(self, x, capacity=None):
            return super().begin_cache(x, capacity)

    class Model(DilutionLM):
        def prefill(self, idx, capacity=None):
            return super().prefill(idx, capacity)

    cfg = LMConfig(vocab_size=32, n_layers=2, d_model=64, n_heads=4, attention="softmax")
    plain, model = DilutionLM(cfg), Model(cfg)
    model.h[0] = Layer(cfg, "softmax")
    for block in model.h:
        block.attn = Attention(cfg)
    model.load_state_dict(plain.state_dict())
    idx = torch.arange(6)[None]
    assert torch.equal(model.generate(idx, 4), plain.generate(idx, 4))
