"""What mm_lora_backward_f32 refuses, before any launch (runs without a GPU)."""

from __future__ import annotations

import ctypes

import pytest

from mmfp4 import _lib

P = ctypes.c_void_p(16)


@pytest.mark.parametrize("kw,msg", [
    ({"mul": ctypes.c_void_p(2)}, "aligned"), ({"base": ctypes.c_void_p(6)}, "aligned"),
    ({"dx": ctypes.c_void_p(1)}, "aligned"), ({"T": 0}, "no tokens"), ({"grad": 2}, "grad_type"),
    ({"L": 1025}, "at most 1024"), ({"K": 0}, "bad shape"), ({}, "workspace")])
def test_refusals(kw, msg):
    o = {"mul": P, "base": None, "dx": P, "T": 4, "grad": 0, "L": 2, "K": 64, **kw}
    with pytest.raises(ValueError, match=f"mm_lora_backward_f32.*{msg}"):
        _lib.call("mm_lora_backward_f32", P, o["mul"], P, P, P, P, 0, None, ctypes.c_float(1.0),
                  o["base"], o["dx"], P, P, o["grad"], o["T"], o["K"], 64, 8, o["L"], None, 0, None)
