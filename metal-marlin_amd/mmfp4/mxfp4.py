"""Microscaled 4-bit floating point (MXFP4, the OCP microscaling format): E2M1 codes with one
power of two per block of 32 values along K.  Unlike the FP4 products of kernels.py, whose groups
have fp16 scales and whose activations stay fp16 (metal_marlin/kernels_core.py:1830-1937), both
sides of these products are 4 bits wide, which the matrix cores multiply as they are.

  words  int32 (or uint32) [*, K/8]   row-packed as MMFP4Linear's: value 8j+i in bits 4i..4i+3
  scales uint8 [*, K/32]              E8M0: c stands for 2^(c - 127), 255 for a block of NaNs
                                      (torch.float8_e8m0fnu tensors are taken as well)

A block's scale is 2^(floor(log2(its largest magnitude)) - 2), at least 2^-127; its values are
rounded to nearest, ties to even, and saturate at 6 times the scale; a block that holds a NaN or
an infinity becomes NaNs.
"""

from __future__ import annotations

import torch

from . import _lib
from .backward import _TYPES, _type, on_device, plain

__all__ = ["mxfp4_quantize", "mxfp4_dequantize", "mxfp4_gemm"]

BLOCK = 32


def _scales(t: torch.Tensor, name: str = "scales") -> torch.Tensor:
    e8m0 = getattr(torch, "float8_e8m0fnu", None)
    if e8m0 is not None and t.dtype == e8m0:
        t = t.view(torch.uint8)
    if t.dtype != torch.uint8:
        raise TypeError(f"{name} must be uint8 (E8M0 codes), got {t.dtype}")
    return t


def _weights(words: torch.Tensor, scales: torch.Tensor, dims: int | None = None,
             name: str = "words") -> tuple[torch.Tensor, torch.Tensor]:
    """The checked pair: words [*, K/8] and scales [*, K/32] of as many axes as `dims`."""
    if words.dtype not in (torch.int32, torch.uint32):
        raise TypeError(f"{name} must be int32/uint32, got {words.dtype}")
    scales = _scales(scales, f"scales of {name}")
    if words.dim() == 0 or (dims is not None and words.dim() != dims):
        raise ValueError(f"{name} must have {dims or 'at least 1'} axes, got {tuple(words.shape)}")
    if words.shape[-1] == 0 or words.shape[-1] % 4 != 0:
        raise ValueError(f"{name} shape {tuple(words.shape)}: K={8 * words.shape[-1]} must be a "
                         f"positive multiple of {BLOCK}")
    if tuple(scales.shape) != (*words.shape[:-1], words.shape[-1] // 4):
        raise ValueError(f"scales shape {tuple(scales.shape)} != "
                         f"{(*words.shape[:-1], words.shape[-1] // 4)} for {name} "
                         f"{tuple(words.shape)}")
    return words, scales


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [*, K] fp16, bf16 or fp32, K % 32 == 0 -> words int32 [*, K/8], scales uint8 [*, K/32].
    quantize_fp4 is its counterpart for groups with fp16 scales."""
    dev = _lib.require_device(x)
    _type("x", x.dtype)
    out = _lib.fast("mx_quantize", x, x.detach())
    if out is not None:
        return out
    if x.dim() == 0 or x.shape[-1] == 0 or x.shape[-1] % BLOCK != 0:
        raise ValueError(f"x shape {tuple(x.shape)}: the last axis must be a positive multiple of "
                         f"{BLOCK}")
    K = x.shape[-1]
    with on_device(dev):
        a = plain(x.detach())
        words = torch.empty((*x.shape[:-1], K // 8), dtype=torch.int32, device=dev)
        scales = torch.empty((*x.shape[:-1], K // BLOCK), dtype=torch.uint8, device=dev)
        _lib.call("mm_mxfp4_quantize", _lib.ptr(a), _TYPES[a.dtype], a.numel() // K, K,
                  _lib.ptr(words), _lib.ptr(scales), _lib.stream_of(a))
    return words, scales


def mxfp4_dequantize(words: torch.Tensor, scales: torch.Tensor,
                     dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values of words [*, K/8] with scales [*, K/32] -> [*, K]: exact in bf16 and fp32 but
    for what lies beyond their largest value; rounded to nearest in fp16."""
    dev = _lib.require_device(words, scales)
    _type("dtype", dtype)
    out = _lib.fast("mx_dequantize", words, words, scales, _TYPES[dtype])
    if out is not None:
        return out
    words, scales = _weights(words, scales)
    K = 8 * words.shape[-1]
    with on_device(dev):
        w, s = plain(words), scales.contiguous()
        out = torch.empty((*words.shape[:-1], K), dtype=dtype, device=dev)
        _lib.call("mm_mxfp4_dequantize", _lib.ptr(w), _lib.ptr(s), out.numel() // K, K,
                  _lib.ptr(out), _TYPES[dtype], _lib.stream_of(w))
    return out


def _gemm(x: torch.Tensor, words: torch.Tensor, scales: torch.Tensor,
          out_dtype: torch.dtype | None) -> torch.Tensor:
    dev = _lib.require_device(x, words, scales)
    _type("x", x.dtype)
    dtype = out_dtype or x.dtype
    _type("out_dtype", dtype)
    out = _lib.fast("mx_gemm", x, x, words, scales, _TYPES[dtype])
    if out is not None:
        return out
    words, scales = _weights(words, scales, 2)
    N, K = words.shape[0], 8 * words.shape[1]
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x shape {tuple(x.shape)} must end in K={K}")
    with on_device(dev):
        a = plain(x.reshape(-1, K))
        w, s = plain(words), scales.contiguous()
        M = a.shape[0]
        out = torch.empty((*x.shape[:-1], N), dtype=dtype, device=dev)
        if out.numel() == 0:
            return out
        stream = _lib.raw_stream(dev.index)
        ws = _lib.workspace_on(dev.index, stream,
                               _lib.load().mm_mxfp4_gemm_workspace_bytes(M, N, K))
        _lib.call("mm_mxfp4_gemm", _lib.ptr(a), _TYPES[a.dtype], _lib.ptr(w), _lib.ptr(s),
                  _lib.ptr(out), _TYPES[dtype], M, N, K, _lib.ptr(ws), ws.numel(), stream)
    return out


def mxfp4_gemm(x: torch.Tensor, words: torch.Tensor, scales: torch.Tensor,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """q(x) @ W^T [*, N] in x's type or out_dtype: x [*, K] fp16, bf16 or fp32 is quantized as
    mxfp4_quantize does, W [N, K] is given so (words [N, K/8], scales [N, K/32]); fp32 sums,
    rounded once."""
    return _gemm(x, words, scales, out_dtype)
