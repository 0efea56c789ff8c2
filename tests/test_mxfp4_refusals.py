"""What the MXFP4 entry points refuse, before anything reaches a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mmfp4
from mmfp4 import _lib, mxfp4

P = ctypes.c_void_p(4096)


@pytest.mark.parametrize("name,args,msg", [
    ("mm_mxfp4_quantize", (P, 1, 4, 48, P, P, None), "multiple of 32"),
    ("mm_mxfp4_quantize", (P, 1, -1, 64, P, P, None), "rows=-1"),
    ("mm_mxfp4_quantize", (P, 3, 4, 64, P, P, None), "type 3"),
    ("mm_mxfp4_quantize", (ctypes.c_void_p(4104), 1, 4, 64, P, P, None), "aligned"),
    ("mm_mxfp4_quantize", (None, 1, 4, 64, P, P, None), "null"),
    ("mm_mxfp4_dequantize", (P, P, 4, 0, P, 1, None), "multiple of 32"),
    ("mm_mxfp4_dequantize", (P, P, 4, 64, P, -1, None), "type -1"),
    ("mm_mxfp4_dequantize", (P, P, 4, 64, ctypes.c_void_p(4098), 1, None), "aligned"),
    ("mm_mxfp4_gemm", (P, 1, P, P, P, 1, 4, 64, 40, None, 0, None), "multiple of 32"),
    ("mm_mxfp4_gemm", (P, 5, P, P, P, 1, 4, 64, 64, None, 0, None), "type 5"),
    ("mm_mxfp4_gemm", (P, 1, P, P, P, 7, 4, 64, 64, None, 0, None), "7"),
    ("mm_mxfp4_gemm", (P, 1, ctypes.c_void_p(8), P, P, 1, 4, 64, 64, None, 0, None), "aligned"),
    ("mm_mxfp4_gemm", (P, 1, P, P, P, 1, 4, 0, 64, None, 0, None), "N=0"),
    ("mm_mxfp4_gemm", (P, 1, P, P, P, 1, 400, 64, 64, None, 0, None), "workspace"),
])
def test_entry_points_refuse(name, args, msg):
    with pytest.raises(ValueError, match=msg):
        _lib.call(name, *args)


def test_nothing_to_do_is_no_error():
    _lib.call("mm_mxfp4_quantize", None, 1, 0, 64, None, None, None)
    _lib.call("mm_mxfp4_dequantize", None, None, 0, 64, None, 1, None)
    _lib.call("mm_mxfp4_gemm", None, 1, None, None, None, 1, 0, 64, 64, None, 0, None)


def test_host_tensors_and_types_are_refused():
    w, s = torch.zeros(8, 8, dtype=torch.int32), torch.zeros(8, 2, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="GPU"):
        mmfp4.mxfp4_quantize(torch.zeros(2, 64))
    with pytest.raises(RuntimeError, match="GPU"):
        mmfp4.mxfp4_dequantize(w, s)
    with pytest.raises(RuntimeError, match="GPU"):
        mmfp4.mxfp4_gemm(torch.zeros(2, 64), w, s)
    with pytest.raises(TypeError):
        mmfp4.mxfp4_gemm([1.0], w, s)


@pytest.mark.parametrize("words,scales,error", [
    (torch.zeros(8, 8), torch.zeros(8, 2, dtype=torch.uint8), TypeError),
    (torch.zeros(8, 8, dtype=torch.int32), torch.zeros(8, 2, dtype=torch.float16), TypeError),
    (torch.zeros(8, 6, dtype=torch.int32), torch.zeros(8, 1, dtype=torch.uint8), ValueError),
    (torch.zeros(8, 8, dtype=torch.int32), torch.zeros(2, 8, dtype=torch.uint8), ValueError),
    (torch.zeros(8, 8, dtype=torch.int32), torch.zeros(8, 3, dtype=torch.uint8), ValueError),
    (torch.zeros(64, dtype=torch.int32), torch.zeros(16, dtype=torch.uint8), ValueError),
])
def test_weights_are_checked(words, scales, error):
    with pytest.raises(error):
        mxfp4._weights(words, scales, 2)
