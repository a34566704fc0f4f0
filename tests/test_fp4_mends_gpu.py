"""Calls on 4-bit caches that are refused before they write, and calls beside them that are taken, on the GPU."""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref
from dilution import cache, kernels
from gpu_helpers import needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]


def _state(b, h, cap, d, seed):
    g = torch.Generator().manual_seed(seed)
    caches = [kernels.Fp4Rows(*(x.cuda() for x in ref.quantise(torch.randn(b, h, cap, d, generator=g)))) for _ in range(2)]
    return torch.randn(b, h, 1, d, generator=g).cuda(), *caches, torch.zeros(b, h, cap, device="cuda")


def test_a_workspace_off_its_alignment_is_refused():
    b, h, top, d = 1, 2, 9000, 64
    q, kc, vc, com = _state(b, h, top, d, 1)
    need = kernels.decode_fp4_workspace(b, h, top, d, "cuda").numel()
    buf = torch.empty(need + 64, dtype=torch.uint8, device="cuda")
    length = torch.tensor([top], device="cuda")
    for off in (1, 4, 8):
        with pytest.raises(ValueError, match="16-byte aligned"):
            kernels.decode_step_fp4_device_length(q, kc, vc, com, length, top, workspace=buf[off:])
    assert not com.any()
    want = com.clone()
    out = kernels.dilution_decode_step_fp4(q, kc, vc, want, top)
    got = kernels.decode_step_fp4_device_length(q, kc, vc, com, length, top, workspace=buf[16:])
    assert torch.equal(got, out) and torch.equal(com, want)
    # where one launch does the step no workspace is used
    short = torch.tensor([300], device="cuda")
    kernels.decode_step_fp4_device_length(q, kc, vc, com, short, 300, workspace=buf[1:])


def test_one_position_is_appended():
    q, kc, vc, com = _state(1, 2, 8, 64, 2)
    c = {"k": kc, "v": vc, "len": 5, "committed": com}
    before = [x.clone() for x in (*kc, *vc)]
    for rows in (0, 2, 3):
        x = torch.ones(1, 2, rows, 64, device="cuda")
        with pytest.raises(ValueError, match="one new position"):
            cache.append_kv(c, x, x)
    assert c["len"] == 5 and all(torch.equal(x, y) for x, y in zip((*kc, *vc), before))
    assert cache.append_kv(c, q, -q) == 6 == c["len"]
    k, v = kernels.dilution_fp4_read(kc, vc, 5, 1, torch.float32)
    want = ref.values(*ref.quantise(q)).float()
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), -want)
