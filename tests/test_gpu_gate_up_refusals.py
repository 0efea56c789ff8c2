"""Shapes that the gated block's backward pass refuses, whichever path takes the call."""

from __future__ import annotations

import pytest
import torch

import mmfp4

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dh,kept", [((2, 3), (3, 2)), ((6,), (2, 3)), ((2, 3), (6,)),
                                     ((4,), (5,)), ((2, 0), (0, 2))])
def test_leading_axes(dh, kept, dtype):
    N, K, g = 64, 128, 64
    w = (torch.randn((N, K), device=DEV) * 0.05).half()
    mats = mmfp4.quantize_fp4(w, group_size=g) * 2
    d = torch.zeros((*dh, N), dtype=dtype, device=DEV)
    gu = torch.zeros((*kept, 2 * N), dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="gate_up shape"):
        mmfp4.fused_gate_up_swiglu_backward(d, gu, *mats, g)
    gu = torch.zeros((*dh, 2 * N), dtype=torch.float16, device=DEV)
    assert mmfp4.fused_gate_up_swiglu_backward(d, gu, *mats, g).shape == (*dh, K)
