"""Autograd over the quantized products: gradients of the input through frozen 4-bit weights,
and of low-rank adapters.  The layers (QuantizedLinear, MarlinLinear, MMFP4Linear, LoRALinear),
the products (marlin_gemm_fp4, marlin_gemm_int4, mmfp4_gemm_rowpacked, mmfp4_fused_qkv and what
is made of them), fused_gate_up_swiglu and lora_add use these by themselves where an operand
requires a gradient; calls that need none take the same path as ever.  They are differentiable
once: a gradient of a gradient is an error, not a silent zero.

A backward pass may be captured into a graph.  torch then refuses, by ending the process, one
thing that a caller cannot see: a leaf whose gradient accumulator belongs to another stream
because an eager graph of that leaf is still alive.  refuse_foreign_leaf raises before that.
"""

from __future__ import annotations

from collections.abc import Callable

import torch
from torch.autograd.function import once_differentiable

from . import _lib, adapters, backward, kernels

__all__ = ["linear", "marlin_gemm", "rowpacked_gemm", "gate_up_swiglu", "FusedQKV", "GateUp",
           "LoraAdd", "LoraLinear"]


def refuse_foreign_leaf(*tensors: torch.Tensor | None) -> None:
    """Under graph capture, raises for a leaf behind `tensors` whose gradient accumulator lives
    on another stream than the captured one."""
    b = _lib.binding()
    if b is None or not torch.cuda.is_current_stream_capturing():
        return
    for t in _leaves(tensors):
        stream = b.accumulator_stream(t)
        if stream >= 0 and stream != torch.cuda.current_stream(t.device).stream_id:
            raise RuntimeError(
                "backward under graph capture: a leaf's gradient accumulator belongs to "
                "another stream, because a graph built there is still alive. Drop it (del "
                "its outputs) before capturing, or build it on the capture stream too")


def _leaves(tensors):
    """The leaves on the device that gradients of `tensors` will reach."""
    seen, nodes = set(), []
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.requires_grad:
            if t.is_leaf:
                yield t
            else:
                nodes.append(t.grad_fn)
    while nodes:
        node = nodes.pop()
        if node is None or node in seen:
            continue
        seen.add(node)
        leaf = getattr(node, "variable", None)
        if isinstance(leaf, torch.Tensor) and leaf.is_cuda:
            yield leaf
        nodes += [n for n, _ in node.next_functions]


def wants_grad(*tensors: torch.Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(
        isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


class _Linear(torch.autograd.Function):
    """y = forward(x) as it comes or in x's type, dx = input_grad(dy); neither depends on
    anything trained."""

    @staticmethod
    def forward(ctx, x, product, input_grad, cast):
        refuse_foreign_leaf(x)
        ctx.input_grad, ctx.dtype, ctx.shape = input_grad, x.dtype, x.shape
        y = product(x)
        y = y.to(x.dtype) if cast else y
        # a view (columns of a padded product) could not be changed in place, as a bias is added
        return y.clone() if y._is_view() else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return ctx.input_grad(dy, ctx.dtype).view(ctx.shape), None, None, None


def linear(x: torch.Tensor, product: Callable, input_grad: Callable) -> torch.Tensor:
    """product(x) in x's type, differentiable in x: input_grad(dy, dtype) is its gradient."""
    if wants_grad(x):
        return _Linear.apply(x, product, input_grad, True)
    return product(x).to(x.dtype)


def marlin_gemm(kind: str, A: torch.Tensor, B_packed: torch.Tensor, scales: torch.Tensor,
                zeros: torch.Tensor | None, group_size: int) -> torch.Tensor:
    """marlin_gemm_fp4 / marlin_gemm_int4, differentiable in A."""
    def input_grad(dy, dtype):
        if kind == "fp4":
            return backward.marlin_gemm_fp4_backward(dy, B_packed, scales, group_size, dtype)
        return backward.marlin_gemm_int4_backward(dy, B_packed, scales, zeros, group_size, dtype)
    return _Linear.apply(A, lambda x: kernels._gemm(kind, x, B_packed, scales, zeros, group_size),
                         input_grad, False)


def rowpacked_gemm(A: torch.Tensor, B_rows: torch.Tensor, scales: torch.Tensor,
                   group_size: int) -> torch.Tensor:
    """mmfp4_gemm_rowpacked, differentiable in A."""
    return _Linear.apply(
        A, lambda x: kernels.mmfp4_gemm_rowpacked(x, B_rows, scales, group_size),
        lambda dy, dt: backward.mmfp4_gemm_rowpacked_backward(dy, B_rows, scales, group_size, dt),
        False)


class FusedQKV(torch.autograd.Function):
    """mmfp4_fused_qkv, differentiable in A: the three gradients meet in one product."""

    @staticmethod
    def forward(ctx, A, group_size, *weights):
        refuse_foreign_leaf(A)
        ctx.save_for_backward(*weights)
        ctx.group_size, ctx.dtype, ctx.shape = group_size, A.dtype, A.shape
        out = kernels.mmfp4_fused_qkv(A, *weights, group_size)
        return tuple(t.clone() if t._is_view() else t for t in out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk, dv):
        dx = backward.mmfp4_fused_qkv_backward(dq, dk, dv, *ctx.saved_tensors, ctx.group_size,
                                               out_dtype=ctx.dtype)
        return (dx.view(ctx.shape), None, *[None] * 6)


class GateUp(torch.autograd.Function):
    """fused_gate_up_swiglu, its h as it comes or in x's type; h is differentiable in x, what is
    kept is not."""

    @staticmethod
    def forward(ctx, x, gate_packed, gate_scales, up_packed, up_scales, group_size, row_packed,
                cast):
        refuse_foreign_leaf(x)
        h, gate_up = backward.fused_gate_up_swiglu(x, gate_packed, gate_scales, up_packed,
                                                   up_scales, group_size, row_packed)
        ctx.save_for_backward(gate_up, gate_packed, gate_scales, up_packed, up_scales)
        ctx.group_size, ctx.row_packed, ctx.dtype = group_size, row_packed, x.dtype
        ctx.mark_non_differentiable(gate_up)
        return h.to(x.dtype) if cast else h, gate_up

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, _):
        gate_up, *weights = ctx.saved_tensors
        dx = backward.fused_gate_up_swiglu_backward(dh, gate_up, *weights, ctx.group_size,
                                                    ctx.row_packed, out_dtype=ctx.dtype)
        return (dx, *[None] * 7)


def gate_up_swiglu(x: torch.Tensor, gate_packed: torch.Tensor, gate_scales: torch.Tensor,
                   up_packed: torch.Tensor, up_scales: torch.Tensor, group_size: int = 128,
                   row_packed: bool = False) -> torch.Tensor:
    """silu(x @ Wg) * (x @ Wu) in x's type, differentiable in x: fused_gate_up_swiglu and its
    backward pass as one differentiable call."""
    return GateUp.apply(x, gate_packed, gate_scales, up_packed, up_scales, group_size,
                        row_packed, True)[0]


class LoraAdd(torch.autograd.Function):
    """lora_add, differentiable in base, x, lora_a and lora_b."""

    @staticmethod
    def forward(ctx, base, x, lora_a, lora_b, adapter_ids, scaling):
        refuse_foreign_leaf(base, x, lora_a, lora_b)
        ctx.save_for_backward(x, lora_a, lora_b, adapter_ids,
                              scaling if isinstance(scaling, torch.Tensor) else None)
        ctx.scaling = scaling
        ctx.base_dtype = base.dtype
        return adapters._add(base, x, lora_a, lora_b, adapter_ids, scaling)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, a, b, ids, scaling = ctx.saved_tensors
        dx = da = db = None
        if any(ctx.needs_input_grad[1:4]):
            dx, da, db = adapters.lora_backward(dy.contiguous(), x, a, b, ids,
                                                ctx.scaling if scaling is None else scaling)
        return dy.to(ctx.base_dtype), dx, da, db, None, None


def _column_sums(t: torch.Tensor) -> torch.Tensor:
    """[M, N] -> [N] in fp32.  At most 128 rows at a time: sums of more are shared out over
    blocks, whose counters torch clears in a way that a graph must not replay."""
    while t.shape[0] > 128:
        n = t.shape[0] // 128 * 128
        blocks = t[:n].view(-1, 128, t.shape[1]).sum(1, dtype=torch.float32)
        t = torch.cat([blocks, t[n:].float()])
    return t.sum(0, dtype=torch.float32)


class LoraLinear(torch.autograd.Function):
    """A layer and its adapters in one node: the layer's gradient of x, of x's type, is the
    dx_base that the adapters' is added to in fp32.  `bias` is the layer's, for its gradient."""

    @staticmethod
    def forward(ctx, x, lora_a, lora_b, adapter_ids, scaling, layer, bias):
        refuse_foreign_leaf(x, lora_a, lora_b, bias)
        ctx.save_for_backward(x, lora_a, lora_b, adapter_ids,
                              scaling if isinstance(scaling, torch.Tensor) else None)
        ctx.scaling, ctx.layer = scaling, layer
        ctx.bias_dtype = None if bias is None else bias.dtype
        return adapters._add(layer(x), x, lora_a, lora_b, adapter_ids, scaling).to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, a, b, ids, scaling = ctx.saved_tensors
        dy = dy.contiguous()
        dx = da = db = dbias = None
        if any(ctx.needs_input_grad[:3]):
            base = ctx.layer.input_grad(dy, x.dtype) if ctx.needs_input_grad[0] else None
            dx, da, db = adapters.lora_backward(dy, x, a, b, ids,
                                                ctx.scaling if scaling is None else scaling,
                                                dx_base=base)
        if ctx.needs_input_grad[6]:
            dbias = _column_sums(dy.view(-1, dy.shape[-1])).to(ctx.bias_dtype)
        return (dx if ctx.needs_input_grad[0] else None), da, db, None, None, None, dbias
