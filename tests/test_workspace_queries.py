"""The workspace queries at sizes that no call takes."""

from __future__ import annotations

import pytest
import torch

from dilution import _hip, kernels
from gpu_helpers import needs_gpu


@pytest.mark.parametrize("dtype,precision", [(0, 0), (0, 1), (1, 2), (2, 2)])
@pytest.mark.parametrize("d", [16, 64, 256])
def test_queries_without_slices_or_rows_return(d, dtype, precision):
    """No slices or no rows: nothing to hold.  (The call itself then refuses the sizes.)"""
    lib = _hip.lib()
    for n, seq in ((0, 20), (-1, 20), (0, 5000), (2, 0), (2, -4), (0, 0)):
        assert lib.dil_forward_workspace_bytes(n, seq, d, dtype, precision, 1) == 0
        assert lib.dil_prefill_workspace_bytes(n, seq, 0, d, dtype, precision) == 0
        assert lib.dil_tree_workspace_bytes(n, max(seq, 0), 0 if n > 0 else 4, d, dtype) == 0
        assert lib.dil_evict_workspace_bytes(n, seq, 1) == 0
    assert lib.dil_prefill_workspace_bytes(2, 20, -1, d, dtype, precision) == 0


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_calls_without_slices(dtype):
    """A forward of no slices has nothing to launch; a prefill chunk refuses them."""
    q = torch.zeros(0, 2, 40, 64, dtype=dtype, device="cuda")
    com = torch.zeros(0, 2, 40, device="cuda")
    for precision in ("ieee", "bf16"):
        assert kernels.dilution_attention_forward(q, q, q, dot_precision=precision).shape == (0, 2, 40, 64)
        with pytest.raises(RuntimeError, match="invalid shape"):
            kernels.dilution_prefill_chunk(q, q, q, com, 0, dot_precision=precision)
