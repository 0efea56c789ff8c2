"""Counts that a launch cannot hold (2^32 threads, blocks that 31 bits count) are refused before
anything reaches a GPU."""

from __future__ import annotations

import ctypes

import pytest

from mmfp4 import _lib

P = ctypes.c_void_p(4096)
MUCH = 1 << 62
TOP = (1 << 31) - 1


@pytest.mark.parametrize("name,args", [
    ("mm_mxfp4_quantize", (P, 1, 1 << 31, 64, P, P, None)),
    ("mm_mxfp4_quantize", (P, 0, 1 << 60, 1 << 30, P, P, None)),
    ("mm_mxfp4_dequantize", (P, P, 1 << 31, 64, P, 1, None)),
    ("mm_mxfp4_gemm", (P, 1, P, P, P, 1, 1, 1 << 29, 32, P, MUCH, None)),
    ("mm_mxfp4_gemm", (P, 1, P, P, P, 1, 30, TOP, 32, P, MUCH, None)),
    ("mm_mxfp4_gemm", (P, 1, P, P, P, 1, 1 << 28, 64, 32, P, MUCH, None)),
    ("mm_mxfp4_gemm", (P, 1, P, P, P, 1, TOP, 64, 32, P, MUCH, None)),
    ("mm_mxfp4_gemm", (P, 1, P, P, P, 1, 1 << 20, 1 << 28, 32, P, MUCH, None)),
    ("mm_mxfp4_gemm_backward", (P, 1, 8, P, P, P, 1, TOP, 8, 128, P, MUCH, None)),
    ("mm_mxfp4_gemm_backward", (P, 1, 8, P, P, P, 1, TOP - 127, 8, 128, P, MUCH, None)),
    ("mm_mxfp4_gemm_backward", (P, 1, 8, P, P, P, 1, 1 << 24, 8, 1 << 20, P, MUCH, None)),
    ("mm_moe_route", (P, 0, None, TOP, 8, 2, 0, 1, 1, 1, 1.0, P, P, None)),
    ("mm_moe_route", (P, 0, None, 1 << 28, 8, 2, 0, 1, 1, 1, 1.0, P, P, None)),
    ("mm_moe_route", (P, 0, None, 1 << 26, 512, 2, 0, 1, 1, 1, 1.0, P, P, None)),
    ("mm_moe_route_backward", (P, P, 0, P, TOP, 8, 2, 0, 1, 1.0, P, None)),
    ("mm_moe_route_backward", (P, P, 0, P, 1 << 26, 512, 2, 0, 1, 1.0, P, None)),
])
def test_too_many(name, args):
    with pytest.raises(ValueError, match="too (many|large)"):
        _lib.call(name, *args)
