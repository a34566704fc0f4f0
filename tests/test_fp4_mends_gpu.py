"""Calls on 4-bit caches that are refused before they write, and calls beside them that are taken, on the GPU."""

from __future__ import annotations

import pytest
import torch

import fp4_reference as ref
from dilution import kernels
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
