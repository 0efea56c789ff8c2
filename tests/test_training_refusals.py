"""What the input gradients, the kept gate/up block and the adapters refuse, before any launch
(runs without a GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mmfp4
from mmfp4 import _lib

P16 = ctypes.c_void_p(16)


def table(*v):
    return (ctypes.c_void_p * len(v))(*v)


def ints(*v):
    return (ctypes.c_int * len(v))(*v)


def backward(nmat=1, N=(64,), ldc=(64,), layout=0, out_type=1, M=4, K=64, g=32, z=None, a=16,
             ws=None, nbytes=0):
    n = len(N)
    _lib.call("mm_gemm_backward", table(*[a] * n), ints(*ldc), None, nmat, table(*[16] * n),
              table(*[16] * n), z, ints(*N), layout, P16, out_type, M, K, g, ws, nbytes, None)


@pytest.mark.parametrize("kw,msg", [
    ({"nmat": 0}, "nmat"), ({"nmat": 4, "N": (64,) * 4, "ldc": (64,) * 4}, "nmat"),
    ({"N": (60,)}, "multiple of 8"), ({"N": (0,)}, "multiple of 8"), ({"ldc": (56,)}, "ldc"),
    ({"ldc": (68,)}, "ldc"), ({"layout": 2}, "layout"), ({"out_type": 3}, "out_type"),
    ({"K": 60}, "divisible by 8"), ({"K": 72, "layout": 1, "g": 8}, "divisible by 32"),
    ({"g": 12}, "group_size"), ({"g": 48}, "group_size"), ({"a": 8}, "aligned"),
    ({"layout": 1, "z": table(16)}, "zero points"), ({"M": -1}, "bad shape"),
    ({"ldc": (1 << 23,)}, "too long"), ({"M": 1 << 23}, "too large"),
    ({"M": 4, "K": 256, "N": (65536,), "ldc": (65536,)}, "workspace"),
])
def test_backward_product(kw, msg):
    with pytest.raises(ValueError, match=msg):
        backward(**kw)


def test_other_entry_points():
    with pytest.raises(ValueError, match="type"):
        _lib.call("mm_grad_rows", P16, 3, P16, P16, 1, 8, None)
    with pytest.raises(ValueError, match="bad shape"):
        _lib.call("mm_grad_rows", P16, 1, P16, P16, 1, 12, None)
    with pytest.raises(ValueError, match="aligned"):
        _lib.call("mm_swiglu_grad", ctypes.c_void_p(2), 1, P16, P16, P16, 1, 8, None)
    with pytest.raises(ValueError, match="layout"):
        _lib.call("mm_fp4_gate_up_keep", P16, P16, P16, P16, P16, P16, P16, 2, 4, 64, 64, 32,
                  None, 0, None)
    with pytest.raises(ValueError, match="divisible by 8"):
        _lib.call("mm_fp4_gate_up_keep", P16, P16, P16, P16, P16, P16, P16, 0, 4, 60, 64, 32,
                  None, 0, None)


def lora(T=4, K=64, N=64, r=8, L=2, type=1, base_type=1, ids=P16, ids64=0, out=P16, ws=None,
         base=ctypes.c_void_p(32)):
    _lib.call("mm_lora_add", P16, type, base, base_type, out, P16, P16, ids, ids64, None,
              ctypes.c_float(1.0), T, K, N, r, L, ws, 0, None)


@pytest.mark.parametrize("kw,msg", [
    ({"type": 0}, "type"), ({"base_type": 2}, "base_type"), ({"K": 0}, "bad shape"),
    ({"r": 0}, "bad shape"), ({"L": 0}, "bad shape"), ({"T": -1}, "bad shape"),
    ({"ids": None}, "need ids"), ({"L": 1025}, "at most 1024"), ({"ids64": 2}, "ids64"),
    ({"r": 5000}, "too large"), ({"r": 4096, "K": 1 << 20}, "too large"),
    ({"r": 4096, "N": 1 << 20}, "too large"), ({"type": 2, "base": P16}, "in place"), ({}, "workspace"),
])
def test_adapters(kw, msg):
    with pytest.raises(ValueError, match=msg):
        lora(**kw)


def test_adapters_backward():
    def call(T=4, grad_type=1):
        _lib.call("mm_lora_backward", P16, P16, 1, P16, P16, P16, 0, None, ctypes.c_float(1.0),
                  None, P16, P16, P16, grad_type, T, 64, 64, 8, 2, None, 0, None)
    with pytest.raises(ValueError, match="no tokens"):
        call(T=0)
    with pytest.raises(ValueError, match="grad_type"):
        call(grad_type=2)
    with pytest.raises(ValueError, match="workspace"):
        call()


def test_workspace_sizes():
    lib = _lib.load()
    size = lib.mm_gemm_backward_workspace_bytes
    assert size(1, ints(4096), 4096, 4096) == 65536            # no split
    assert size(1, ints(14336), 1, 4096) > 65536
    assert size(0, ints(1), 1, 1) == 65536
    one = lib.mm_lora_workspace_bytes(1, 4096, 4096, 16, 8, 0)
    assert 65536 < one <= 65536 + 1024
    assert lib.mm_lora_workspace_bytes(4096, 4096, 4096, 16, 8, 1) > \
        lib.mm_lora_workspace_bytes(4096, 4096, 4096, 16, 8, 0) > one


def test_host_tensors_are_refused():
    f = lambda *s: torch.zeros(s, dtype=torch.float16)          # noqa: E731
    w = torch.zeros(8, 64, dtype=torch.int32)
    for call in (lambda: mmfp4.marlin_gemm_fp4_backward(f(1, 64), w, f(2, 64), 32),
                 lambda: mmfp4.marlin_gemm_int4_backward(f(1, 64), w, f(2, 64), f(2, 64), 32),
                 lambda: mmfp4.mmfp4_gemm_rowpacked_backward(f(1, 8), w, f(16, 8), 32),
                 lambda: mmfp4.mmfp4_fused_qkv_backward(f(1, 64), f(1, 64), f(1, 64),
                                                        *[w, f(2, 64)] * 3, 32),
                 lambda: mmfp4.fused_gate_up_swiglu(f(1, 64), w, f(2, 64), w, f(2, 64), 32),
                 lambda: mmfp4.fused_gate_up_swiglu_backward(f(1, 64), f(1, 128), w, f(2, 64), w,
                                                             f(2, 64), 32),
                 lambda: mmfp4.lora_add(f(1, 64), f(1, 64), f(8, 64), f(64, 8)),
                 lambda: mmfp4.lora_backward(f(1, 64), f(1, 64), f(8, 64), f(64, 8))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_layers_are_checked():
    with pytest.raises(TypeError, match="quantized layer"):
        mmfp4.LoRALinear(torch.nn.Linear(8, 8), 4)
    w = mmfp4.MarlinLinear(torch.zeros(8, 64, dtype=torch.int32), torch.zeros(2, 64).half())
    with pytest.raises(ValueError, match="positive"):
        mmfp4.LoRALinear(w, 0)
    m = mmfp4.LoRALinear(w, 4, num_adapters=3, dtype=torch.bfloat16)
    assert m.lora_a.shape == (3, 4, 64) and m.lora_b.shape == (3, 64, 4)
    assert not m.lora_b.any() and m.lora_a.dtype == torch.bfloat16
