"""Low-rank adapters of many requests at once beside a shared quantized projection: the
serving form (one adapter id per token, any mix of requests in a batch), and the gradients
that train them.  The reference has no adapters; its projections
(metal_marlin/quantized_linear.py:36-55, layers/mmfp4_linear.py:549-598) are what they stand
beside: the output of any of them is `base` here.
"""

from __future__ import annotations

import torch

from . import _lib
from .backward import _TYPES, _carried, _pad_to, on_device, plain

__all__ = ["lora_add", "lora_backward"]


def _factors(lora_a: torch.Tensor, lora_b: torch.Tensor):
    """[L, r, K] and [L, N, r] (a single adapter may come without the first axis)."""
    a, b = (t.unsqueeze(0) if t.dim() == 2 else t for t in (lora_a, lora_b))
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or \
            a.numel() == 0 or b.numel() == 0:
        raise ValueError("lora_a must be [adapters, rank, K] and lora_b [adapters, N, rank] (or "
                         f"[rank, K] and [N, rank]), got {tuple(lora_a.shape)} and "
                         f"{tuple(lora_b.shape)}")
    return a, b


def _compute_type(x: torch.Tensor) -> torch.dtype:
    """fp32 is computed as fp16, as the products do."""
    if x.dtype not in _TYPES:
        raise TypeError(f"x must be fp16, bf16 or fp32, got {x.dtype}")
    return torch.float16 if x.dtype == torch.float32 else x.dtype


def _ids(adapter_ids: torch.Tensor | None, lead: torch.Size, adapters: int):
    if adapter_ids is None:
        if adapters != 1:
            raise ValueError(f"{adapters} adapters need adapter_ids")
        return None
    if adapter_ids.is_floating_point() or adapter_ids.dtype in (torch.bool, torch.uint64):
        raise TypeError(f"adapter_ids must be integers, got {adapter_ids.dtype}")
    n = 1
    for d in lead:
        n *= d
    if tuple(adapter_ids.shape) not in (tuple(lead), (n,)):
        raise ValueError(f"adapter_ids shape {tuple(adapter_ids.shape)} != {tuple(lead)}: one id "
                         "per token")
    i = adapter_ids.reshape(-1)
    return (i if i.dtype in (torch.int32, torch.int64) else i.to(torch.int32)).contiguous()


def _scaling(scaling, adapters: int, dev: torch.device):
    """(fp32 tensor or None, factor)."""
    if not isinstance(scaling, torch.Tensor):
        return None, float(scaling)
    if scaling.dim() == 0:
        scaling = scaling.expand(adapters)
    if tuple(scaling.shape) != (adapters,):
        raise ValueError(f"scaling shape {tuple(scaling.shape)} != ({adapters},)")
    if scaling.device != dev:
        raise RuntimeError(f"scaling on {scaling.device}, the activations on {dev}")
    return scaling.to(torch.float32).contiguous(), 1.0


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The addresses of t's first element and of the byte behind its last."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _plain_scaling(scaling):
    return (scaling, 1.0) if isinstance(scaling, torch.Tensor) else (None, float(scaling))


def _add(base, x, lora_a, lora_b, adapter_ids, scaling, out=None):
    if out is None and isinstance(x, torch.Tensor):
        got = _lib.fast("lora_add", x, base, x, lora_a, lora_b, adapter_ids,
                        *_plain_scaling(scaling))
        if got is not None:
            return got
    dev = _lib.require_device(base, x, lora_a, lora_b, adapter_ids, out)
    a, b = _factors(lora_a, lora_b)
    L, r, K = a.shape
    N = b.shape[1]
    dt = _compute_type(x)
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x shape {tuple(x.shape)} must end in K={K}")
    if tuple(base.shape) != (*x.shape[:-1], N):
        raise ValueError(f"base shape {tuple(base.shape)} != {(*x.shape[:-1], N)}")
    ids = _ids(adapter_ids, x.shape[:-1], L)
    if out is not None and (out.shape != base.shape or out.dtype != dt or
                            not out.is_contiguous()):
        raise ValueError(f"out must be contiguous {dt} {tuple(base.shape)}, got {out.dtype} "
                         f"{tuple(out.shape)}")
    if out is not None:
        for name, t in (("base", base), ("x", x), ("lora_a", lora_a), ("lora_b", lora_b)):
            itself = t is base and t.dtype == dt and t.is_contiguous() and \
                t.data_ptr() == out.data_ptr()
            if not itself and _overlap(out, t):
                raise ValueError(f"out shares memory with {name}")
    with on_device(dev):
        st, factor = _scaling(scaling, L, dev)
        xf = x.reshape(-1, K).to(dt).contiguous()
        T = xf.shape[0]
        bf = base.reshape(T, N)
        if bf.dtype not in (torch.float16, dt):
            bf = bf.to(dt)
        bf = bf.contiguous()
        a, b = a.to(dt).contiguous(), b.to(dt).contiguous()
        if out is None:
            out = torch.empty(base.shape, dtype=dt, device=dev)
        if T == 0:
            return out
        stream = _lib.raw_stream(dev.index)
        ws = _lib.workspace_on(dev.index, stream,
                               _lib.load().mm_lora_workspace_bytes(T, K, N, r, L, 0))
        _lib.call("mm_lora_add", _lib.ptr(xf), _TYPES[dt], _lib.ptr(bf), _TYPES[bf.dtype],
                  _lib.ptr(out), _lib.ptr(a), _lib.ptr(b), _lib.ptr(ids),
                  int(ids is not None and ids.dtype == torch.int64), _lib.ptr(st), factor, T, K,
                  N, r, L, _lib.ptr(ws), ws.numel(), stream)
    return out


def lora_add(base: torch.Tensor, x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
             adapter_ids: torch.Tensor | None = None, scaling: float | torch.Tensor = 1.0,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = base[t] + scaling[a] * (x[t] @ lora_a[a]^T) @ lora_b[a]^T, a = adapter_ids[t].

    x [*, K] is the input of a projection and base [*, N] its output (of marlin_gemm_fp4, a
    layer, one of mmfp4_fused_qkv's); lora_a [adapters, rank, K], lora_b [adapters, N, rank]
    (a single adapter may come as [rank, K], [N, rank], without ids).  adapter_ids, one per
    token, int32 or int64: an id outside [0, adapters) means no adapter, and that token's out
    is its base.  scaling: a number, or one per adapter.

    fp16 and bf16: factors of another type are converted to x's; base is fp16, as the products
    return it, or of x's type; out has x's type.  fp32 tokens are computed as fp16, and out is
    fp16, as the products return it.  With `out` (contiguous, of that type; base itself will do)
    the result is written there.  Any number of
    tokens and any width or rank, at most 1024 adapters.  Differentiable in base, x, lora_a and
    lora_b (the products and layers that make a base are differentiable in x as well);
    `lora_backward` is the backward pass as a call."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (base, x, lora_a, lora_b)
                                       if isinstance(t, torch.Tensor)):
        from .autograd import LoraAdd
        if isinstance(scaling, torch.Tensor) and scaling.requires_grad:
            raise ValueError("scaling gets no gradient: pass scaling.detach()")
        if out is not None:
            raise ValueError("out= takes no part in autograd: use torch.no_grad()")
        return LoraAdd.apply(base, x, lora_a, lora_b, adapter_ids, scaling)
    return _add(base, x, lora_a, lora_b, adapter_ids, scaling, out)


def lora_backward(dy: torch.Tensor, x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                  adapter_ids: torch.Tensor | None = None, scaling: float | torch.Tensor = 1.0,
                  dx_base: torch.Tensor | None = None):
    """The gradients of lora_add for dy [*, N]: (dx [*, K], da, db), da and db shaped and typed
    as lora_a and lora_b (zeros for adapters without tokens), dx of x's type.  dx_base, the
    gradient that reached x through the projection itself (marlin_gemm_fp4_backward), is
    added to dx before it is rounded.  fp32 tokens are computed as fp16, and their dx is fp32.
    dy of a wider type than fp16 tokens (or fp32 ones) is carried in fp16 under one power of two
    per token, 11 bits of each value; dy beside bf16 tokens is rounded to bf16.  fp32 factors
    beside fp16 or bf16 tokens get fp32 gradients."""
    if isinstance(x, torch.Tensor):
        got = _lib.fast("lora_backward", x, dy, x, lora_a, lora_b, adapter_ids,
                        *_plain_scaling(scaling), dx_base)
        if got is not None:
            return got
    dev = _lib.require_device(dy, x, lora_a, lora_b, adapter_ids, dx_base)
    a, b = _factors(lora_a, lora_b)
    L, r, K = a.shape
    N = b.shape[1]
    dt = _compute_type(x)
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x shape {tuple(x.shape)} must end in K={K}")
    if tuple(dy.shape) != (*x.shape[:-1], N):
        raise ValueError(f"dy shape {tuple(dy.shape)} != {(*x.shape[:-1], N)}")
    if dx_base is not None and dx_base.shape != x.shape:
        raise ValueError(f"dx_base shape {tuple(dx_base.shape)} != {tuple(x.shape)}")
    ids = _ids(adapter_ids, x.shape[:-1], L)
    with on_device(dev):
        st, factor = _scaling(scaling, L, dev)
        xf, dyf = x.reshape(-1, K).to(dt).contiguous(), dy.reshape(-1, N)
        T = xf.shape[0]
        ac, bc = a.to(dt).contiguous(), b.to(dt).contiguous()
        if T == 0:
            return x.new_empty(x.shape), torch.zeros_like(lora_a), torch.zeros_like(lora_b)
        # where dx is fp32, or dy has a wider range than the tokens
        wide = dt == torch.float16 and (x.dtype == torch.float32 or dy.dtype != dt)
        mul = None
        if wide and dy.dtype != dt:
            dyf = dyf if dyf.dtype in _TYPES else dyf.float()
            dyf, mul = _carried(plain(_pad_to(dyf, N + -N % 8)))
            dyf = dyf[:, :N].contiguous()
        else:
            dyf = dyf.to(dt).contiguous()
        dxt = torch.float32 if wide else dt
        dxb = None if dx_base is None else dx_base.reshape(T, K).to(dxt).contiguous()
        dx = torch.empty((T, K), dtype=dxt, device=dev)
        # factors that are not of the type they are computed in (fp32 masters) get their
        # gradients from the fp32 sums
        gt = dt if lora_a.dtype == lora_b.dtype == dt else torch.float32
        da, db = torch.empty_like(ac, dtype=gt), torch.empty_like(bc, dtype=gt)
        stream = _lib.raw_stream(dev.index)
        ws = _lib.workspace_on(dev.index, stream,
                               _lib.load().mm_lora_workspace_bytes(T, K, N, r, L, 1))
        tokens = (_lib.ptr(ac), _lib.ptr(bc), _lib.ptr(ids),
                  int(ids is not None and ids.dtype == torch.int64), _lib.ptr(st), factor,
                  _lib.ptr(dxb), _lib.ptr(dx), _lib.ptr(da), _lib.ptr(db), _TYPES[gt], T, K, N, r,
                  L, _lib.ptr(ws), ws.numel(), stream)
        if wide:
            _lib.call("mm_lora_backward_f32", _lib.ptr(dyf), _lib.ptr(mul), _lib.ptr(xf), *tokens)
        else:
            _lib.call("mm_lora_backward", _lib.ptr(dyf), _lib.ptr(xf), _TYPES[dt], *tokens)
    return (dx.view(x.shape).to(x.dtype), da.view(lora_a.shape).to(lora_a.dtype),
            db.view(lora_b.shape).to(lora_b.dtype))
