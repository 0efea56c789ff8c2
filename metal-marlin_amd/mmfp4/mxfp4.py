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

from . import _lib, kernels
from .backward import _TYPES, _type, on_device, plain

__all__ = ["mxfp4_quantize", "mxfp4_dequantize", "mxfp4_gemm", "mxfp4_gemm_backward",
           "moe_mlp_mxfp4"]

BLOCK = 32


def _scales(t: torch.Tensor, name: str = "scales") -> torch.Tensor:
    e8m0 = getattr(torch, "float8_e8m0fnu", None)
    if e8m0 is not None and t.dtype == e8m0:
        t = t.view(torch.uint8)
    if t.dtype != torch.uint8:
        raise TypeError(f"{name} must be uint8 (E8M0 codes), got {t.dtype}")
    return t


def _count(name: str, n: int) -> int:
    if n >= 1 << 31:
        raise ValueError(f"{name}={n} is too large: at most 2^31 - 1")
    return n


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
    if isinstance(x, torch.Tensor):
        out = _lib.fast("mx_quantize", x, x)
        if out is not None:
            return out
    dev = _lib.require_device(x)
    _type("x", x.dtype)
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
        w, s = plain(words), plain(scales)
        out = torch.empty((*words.shape[:-1], K), dtype=dtype, device=dev)
        _lib.call("mm_mxfp4_dequantize", _lib.ptr(w), _lib.ptr(s), out.numel() // K, K,
                  _lib.ptr(out), _TYPES[dtype], _lib.stream_of(w))
    return out


def _gemm(x: torch.Tensor, words: torch.Tensor, scales: torch.Tensor,
          out_dtype: torch.dtype | None) -> torch.Tensor:
    out = _lib.fast("mx_gemm", x, x, words, scales, -1 if out_dtype is None else _type(
        "out_dtype", out_dtype))
    if out is not None:
        return out
    dev = _lib.require_device(x, words, scales)
    _type("x", x.dtype)
    dtype = out_dtype or x.dtype
    words, scales = _weights(words, scales, 2)
    N, K = _count("N", words.shape[0]), _count("K", 8 * words.shape[1])
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x shape {tuple(x.shape)} must end in K={K}")
    with on_device(dev):
        a = plain(x.reshape(-1, K))
        w, s = plain(words), plain(scales)
        M = _count("rows", a.shape[0])
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
    rounded once.  Differentiable in x, straight through its rounding (mxfp4_gemm_backward)."""
    if isinstance(x, torch.Tensor):
        if kernels._wants_grad(x):
            from . import autograd
            return autograd.mxfp4_product(x, words, scales, out_dtype)
        return _gemm(x, words, scales, out_dtype)
    raise TypeError(f"expected torch.Tensor, got {type(x).__name__}")


def mxfp4_gemm_backward(dy: torch.Tensor, words: torch.Tensor, scales: torch.Tensor,
                        out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dx = dy @ W, the gradient of mxfp4_gemm's input for dy [*, N] -> [*, K] in dy's type or
    out_dtype: x's rounding counts as the identity.  dy (fp16, bf16, or fp32 but for what lies below
    2^-133) and W enter exactly, sums are fp32, rounded once."""
    if not isinstance(dy, torch.Tensor):
        raise TypeError(f"expected torch.Tensor, got {type(dy).__name__}")
    out = _lib.fast("mx_gemm_backward", dy, dy, words, scales, -1 if out_dtype is None else _type(
        "out_dtype", out_dtype))
    if out is not None:
        return out
    dev = _lib.require_device(dy, words, scales)
    _type("dy", dy.dtype)
    dtype = out_dtype or dy.dtype
    words, scales = _weights(words, scales, 2)
    N, K = _count("N", words.shape[0]), _count("K", 8 * words.shape[1])
    if dy.dim() == 0 or dy.shape[-1] != N:
        raise ValueError(f"dy shape {tuple(dy.shape)} must end in N={N}")
    with on_device(dev):
        out = torch.empty((*dy.shape[:-1], K), dtype=dtype, device=dev)
        if out.numel() == 0:
            return out
        if N == 0:
            return out.zero_()
        w, s = plain(words), plain(scales)
        d, pad = dy.reshape(-1, N), -N % (4 if dy.dtype == torch.float32 else 8)
        if pad:                 # rows of whole 16-byte pieces
            d = torch.nn.functional.pad(d, (0, pad))
        d = plain(d)
        M = _count("rows", d.shape[0])
        stream = _lib.raw_stream(dev.index)
        need = _lib.load().mm_mxfp4_gemm_backward_workspace_bytes(M, N, K, _TYPES[d.dtype])
        ws = _lib.workspace_on(dev.index, stream, need)
        _lib.call("mm_mxfp4_gemm_backward", _lib.ptr(d), _TYPES[d.dtype], N + pad,
                  _lib.ptr(w), _lib.ptr(s), _lib.ptr(out), _TYPES[dtype], M, N, K, _lib.ptr(ws),
                  ws.numel(), stream)
    return out


def moe_mlp_mxfp4(hidden: torch.Tensor, gate_up_words: torch.Tensor, gate_up_scales: torch.Tensor,
                  down_words: torch.Tensor, down_scales: torch.Tensor, expert_ids: torch.Tensor,
                  expert_probs: torch.Tensor) -> torch.Tensor:
    """moe_mlp_fp4 on MXFP4 weights (metal_marlin/moe_dispatch.py:1241-1431 per expert, combined
    as :812-925): for hidden [T, H] of fp16, bf16 or fp32 and its experts [T, k] (as moe_route or
    router_softmax_topk give them),
        (g | u) = q(x) @ W_gu[e]^T;  a = q(silu(g) * u);  y = a @ W_dn[e]^T
        out[t] = sum_j p[t, j] * y                        [T, H] in hidden's type
    gate_up_words [E, 2I, H/8] and scales [E, 2I, H/32], the gate's I rows first; down_words
    [E, H, I/8] and scales [E, H, I/32].  silu(g) * u is quantized from its fp32 value.  Ids
    outside [0, E) contribute nothing.  Not differentiable, as the other products of experts: a
    backward pass that reaches its result raises."""
    if kernels._wants_grad(hidden) or kernels._wants_grad(expert_probs):
        from . import autograd
        return autograd.Undifferentiable.apply(
            "moe_mlp_mxfp4", lambda: _moe_mlp(hidden, gate_up_words, gate_up_scales, down_words,
                                              down_scales, expert_ids, expert_probs),
            hidden, expert_probs)
    return _moe_mlp(hidden, gate_up_words, gate_up_scales, down_words, down_scales, expert_ids,
                    expert_probs)


def _moe_mlp(hidden, gate_up_words, gate_up_scales, down_words, down_scales, expert_ids,
             expert_probs) -> torch.Tensor:
    dev = _lib.require_device(hidden, gate_up_words, gate_up_scales, down_words, down_scales,
                              expert_ids, expert_probs)
    _type("hidden", hidden.dtype)
    out = _lib.fast("mx_moe_mlp", hidden, hidden, gate_up_words, gate_up_scales, down_words,
                    down_scales, expert_ids, expert_probs)
    if out is not None:
        return out
    gu, gus = _weights(gate_up_words, gate_up_scales, 3, "gate_up_words")
    dn, dns = _weights(down_words, down_scales, 3, "down_words")
    E, N2, H = gu.shape[0], gu.shape[1], 8 * gu.shape[2]
    I = 8 * dn.shape[2]
    if N2 != 2 * I or tuple(dn.shape[:2]) != (E, H):
        raise ValueError(f"down_words shape {tuple(dn.shape)} != ({E}, {H}, {N2 // 16}) for "
                         f"gate_up_words {tuple(gu.shape)}")
    if hidden.dim() != 2 or hidden.shape[1] != H:
        raise ValueError(f"hidden shape {tuple(hidden.shape)} must be [T, {H}]")
    T = _count("T", hidden.shape[0])
    if expert_ids.dim() != 2 or expert_ids.shape[0] != T or expert_ids.shape[1] == 0 or \
            expert_probs.shape != expert_ids.shape:
        raise ValueError(f"expert_ids {tuple(expert_ids.shape)} and expert_probs "
                         f"{tuple(expert_probs.shape)} must be [{T}, top_k]")
    if expert_ids.is_floating_point() or expert_ids.dtype in (torch.bool, torch.uint64):
        raise TypeError(f"expert_ids must be integers, got {expert_ids.dtype}")
    k = expert_ids.shape[1]
    with on_device(dev):
        x = plain(hidden)
        ids = expert_ids if expert_ids.dtype == torch.int64 else expert_ids.to(torch.int32)
        ids, p = ids.contiguous(), expert_probs.to(torch.float32).contiguous()
        gu, gus, dn, dns = map(plain, (gu, gus, dn, dns))
        out = torch.empty((T, H), dtype=hidden.dtype, device=dev)
        if T == 0:
            return out
        if E == 0:
            return out.zero_()
        need = _lib.load().mm_moe_mlp_mxfp4_scratch_bytes(T, k, E, H, I)
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.call("mm_moe_mlp_mxfp4", _lib.ptr(x), _TYPES[x.dtype], _lib.ptr(ids),
                  int(ids.dtype == torch.int64), _lib.ptr(p), T, k, E, H, I, _lib.ptr(gu),
                  _lib.ptr(gus), _lib.ptr(dn), _lib.ptr(dns), _lib.ptr(scratch), need,
                  _lib.ptr(out), _lib.stream_of(x))
    return out
