"""Routing of tokens to experts with sigmoid or softmax scores, a balance bias and groups, and
its gradient.  router_softmax_topk (metal_marlin/moe_dispatch.py:99-151) is the softmax of all
experts and their top-k alone; its ids and weights and these go into the same grouped products
(group_tokens_by_expert, moe_mlp_fp4, moe_mlp_mxfp4).
"""

from __future__ import annotations

import torch

from . import _lib, autograd
from .backward import _TYPES, _type, on_device

__all__ = ["moe_route", "moe_route_backward"]

_SCORING = {"sigmoid": False, "softmax": True}


def _softmax(scoring: str) -> bool:
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be 'sigmoid' or 'softmax', got {scoring!r}")
    return _SCORING[scoring]


def _tokens(logits: torch.Tensor) -> int:
    """The rows of logits [*, E]."""
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"logits must be [*, num_experts], got {tuple(logits.shape)}")
    T = logits.numel() // logits.shape[-1]
    if T >= 1 << 31:
        raise ValueError(f"{T} tokens are too many: at most 2^31 - 1")
    return T


def _route(logits, top_k, softmax, bias, num_groups, topk_groups, renormalize, scale):
    if isinstance(logits, torch.Tensor) and (bias is None or isinstance(bias, torch.Tensor)):
        out = _lib.fast("moe_route", logits, logits, top_k, softmax, bias, num_groups, topk_groups,
                        renormalize, scale)
        if out is not None:
            return out
    dev = _lib.require_device(logits, bias)
    _type("logits", logits.dtype)
    T = _tokens(logits)
    E = logits.shape[-1]
    if bias is not None and tuple(bias.shape) != (E,):
        raise ValueError(f"bias shape {tuple(bias.shape)} != ({E},)")
    with on_device(dev):
        l = logits.contiguous()
        b = None if bias is None else bias.to(torch.float32).contiguous()
        shape = (*logits.shape[:-1], max(0, top_k))
        ids = torch.empty(shape, dtype=torch.int64, device=dev)
        w = torch.empty(shape, dtype=torch.float32, device=dev)
        _lib.call("mm_moe_route", _lib.ptr(l), _TYPES[l.dtype], _lib.ptr(b), T, E,
                  top_k, int(softmax), num_groups, topk_groups, int(renormalize), scale,
                  _lib.ptr(ids), _lib.ptr(w), _lib.stream_of(l))
    return w, ids


def moe_route(logits: torch.Tensor, top_k: int, *, scoring: str = "sigmoid",
              bias: torch.Tensor | None = None, num_groups: int = 1, topk_groups: int = 1,
              renormalize: bool = True, scale: float = 1.0):
    """logits [*, E] -> (weights fp32 [*, top_k], ids int64 [*, top_k]).

    s = sigmoid(logits) or softmax(logits).  Experts are ranked by s + bias (bias [E], taken as
    fp32, which moves the choice and no weight); with num_groups > 1 only those of the topk_groups
    groups (E / num_groups experts side by side) with the largest sums of their two best s + bias
    are eligible.  That is so without a bias too: where a model ranks its groups by their best
    expert alone, these are not its experts.  The
    weights are scale * s of the chosen, with renormalize divided by (their sum + 1e-20).  Ties go
    to the lower index.  At most 1024 experts, 64 of them chosen, 64 groups, and fewer than 2^26
    tokens (2^28 with up to 256 experts in up to 16 groups).  NaNs rank last; a
    softmax row of nothing but -inf has weights 0.  Differentiable in logits."""
    if isinstance(logits, torch.Tensor) and autograd.wants_grad(logits):
        return autograd.Route.apply(logits, top_k, _softmax(scoring), bias, num_groups,
                                    topk_groups, renormalize, float(scale))
    return _route(logits, top_k, _softmax(scoring), bias, num_groups, topk_groups, renormalize,
                  float(scale))


def moe_route_backward(dweights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, *,
                       scoring: str = "sigmoid", renormalize: bool = True, scale: float = 1.0):
    """The gradient of moe_route's weights: dweights [*, top_k] -> dlogits [*, E] of the logits'
    type, for the logits and ids of the forward pass.  Ids outside [0, E) get nothing."""
    softmax = _softmax(scoring)
    if all(isinstance(t, torch.Tensor) for t in (dweights, logits, ids)):
        out = _lib.fast("moe_route_backward", logits, dweights, logits, ids, softmax, renormalize,
                        float(scale))
        if out is not None:
            return out
    dev = _lib.require_device(dweights, logits, ids)
    _type("logits", logits.dtype)
    T = _tokens(logits)
    if ids.dim() != logits.dim() or ids.shape[:-1] != logits.shape[:-1] or \
            dweights.shape != ids.shape:
        raise ValueError(f"dweights {tuple(dweights.shape)} and ids {tuple(ids.shape)} must be "
                         f"{(*logits.shape[:-1], 'top_k')}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    _type("dweights", dweights.dtype)
    E = logits.shape[-1]
    with on_device(dev):
        l, i = logits.contiguous(), ids.to(torch.int64).contiguous()
        dw = dweights.to(torch.float32).contiguous()
        dl = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        _lib.call("mm_moe_route_backward", _lib.ptr(dw), _lib.ptr(l), _TYPES[l.dtype],
                  _lib.ptr(i), T, E, ids.shape[-1], int(softmax), int(renormalize),
                  float(scale), _lib.ptr(dl), _lib.stream_of(l))
    return dl
