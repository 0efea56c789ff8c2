"""Input gradients of the quantized products, and the gate/up block that keeps what its
backward pass needs.  The 4-bit weights are frozen: what is trained beside them (adapters,
norms, embeddings, soft prompts) needs dA = dC @ W^T through every layer.  The reference
has no backward pass (metal_marlin/quantized_linear.py:36-55 is forward only).

Gradients are fp16, bf16 or fp32, and the result has the gradient's type unless
`out_dtype` says otherwise.  fp16 ones are multiplied as they are; bf16 and fp32 ones, and
those inside the gate/up block, are carried in fp16 under one power of two per row: bf16 ones
exactly and the others to 11 bits, but for what lies 2^-40 below a row's largest value.  The
products are fp16 x fp16 in fp32 sums, and the sum is rounded once.
"""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib, kernels

__all__ = ["marlin_gemm_fp4_backward", "marlin_gemm_int4_backward",
           "mmfp4_gemm_rowpacked_backward", "mmfp4_fused_qkv_backward",
           "fused_gate_up_swiglu", "fused_gate_up_swiglu_backward"]

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _type(name: str, t: torch.dtype) -> int:
    if t not in _TYPES:
        raise TypeError(f"{name} must be fp16, bf16 or fp32, got {t}")
    return _TYPES[t]


def on_device(dev: torch.device):
    """The device's own context where it is not the current one: the default stream's handle
    means the current device."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def plain(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and 16-byte aligned (a copy where it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _pad_to(t: torch.Tensor, n: int, dim: int = 1, value: float = 0) -> torch.Tensor:
    if t.shape[dim] == n:
        return t
    pad = [0, 0] * (t.dim() - 1 - dim) + [0, n - t.shape[dim]]
    return torch.nn.functional.pad(t.view(torch.int32) if t.dtype == torch.uint32 else t, pad,
                                   value=value)


def _words8(words: torch.Tensor, dim: int = 1) -> torch.Tensor:
    """Packed words with N padded to a multiple of 8 (the copy is kept on the tensor)."""
    n = words.shape[dim]
    if n % 8 == 0:
        return plain(kernels._packed(words))
    return plain(_lib.derived(kernels._packed(words), f"pad8_{dim}",
                              lambda t: _pad_to(t, n + -n % 8, dim)))


def _half8(t: torch.Tensor, value: float) -> torch.Tensor:
    n = t.shape[1]
    if n % 8 == 0:
        return plain(kernels._half(t))
    return plain(kernels._half(_lib.derived(t, f"pad8_{value}",
                                            lambda s: _pad_to(s, n + -n % 8, 1, value))))


def _flat(dC: torch.Tensor, N: int, name: str) -> torch.Tensor:
    """[*, N] -> [M, N8], N8 the next multiple of 8."""
    _type(name, dC.dtype)
    if dC.dim() == 0 or dC.shape[-1] != N:
        raise ValueError(f"{name} shape {tuple(dC.shape)} must end in N={N}")
    return plain(_pad_to(dC.reshape(-1, N), N + -N % 8))


def _launch(dC: list[torch.Tensor], ldc: list[int], row_mul: torch.Tensor | None,
            mats: list[tuple], layout: int, K: int, group_size: int,
            dtype: torch.dtype) -> torch.Tensor:
    """mats: (words, scales, zeros or None) with N % 8 == 0.  dC fp16 [M, >= N]."""
    n = len(mats)
    M, dev = dC[0].shape[0], dC[0].device
    out = torch.empty((M, K), dtype=dtype, device=dev)
    if M == 0:
        return out
    Ns = (ctypes.c_int * n)(*[s.shape[1] for _, s, _ in mats])
    table = lambda ts: (ctypes.c_void_p * n)(*[t.data_ptr() for t in ts])   # noqa: E731
    zeros = table([z for _, _, z in mats]) if mats[0][2] is not None else None
    stream = _lib.raw_stream(dev.index)
    need = _lib.load().mm_gemm_backward_workspace_bytes(n, Ns, M, K)
    ws = _lib.workspace_on(dev.index, stream, need)
    _lib.call("mm_gemm_backward", table(dC), (ctypes.c_int * n)(*ldc),
              _lib.ptr(row_mul), n, table([w for w, _, _ in mats]),
              table([s for _, s, _ in mats]), zeros, Ns, layout, _lib.ptr(out), _TYPES[dtype], M,
              K, group_size, _lib.ptr(ws), ws.numel(), stream)
    return out


def _carried(g: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor | None]:
    """fp16 values of g [M, N8] and the rows' factors (None: ones)."""
    if g.dtype == torch.float16:
        return g, None
    M, N = g.shape
    y = torch.empty((M, N), dtype=torch.float16, device=g.device)
    mul = torch.empty(M, dtype=torch.float32, device=g.device)
    _lib.call("mm_grad_rows", _lib.ptr(g), _TYPES[g.dtype], _lib.ptr(y), _lib.ptr(mul), M, N,
              _lib.stream_of(g))
    return y, mul


def _linear(dC: torch.Tensor, words: torch.Tensor, scales: torch.Tensor,
            zeros: torch.Tensor | None, layout: int, K: int, group_size: int,
            out_dtype: torch.dtype | None) -> torch.Tensor:
    dev = _lib.require_device(dC, words, scales, zeros)
    N = scales.shape[1]
    dtype = out_dtype or dC.dtype
    if dtype == dC.dtype:
        out = _lib.fast("linear_backward", dC, dC, words, scales, zeros, bool(layout), group_size)
        if out is not None:
            return out
    _type("out_dtype", dtype)
    with on_device(dev):
        g, mul = _carried(_flat(dC, N, "dC"))
        mat = (_words8(words, 1 - layout), _half8(scales, 1.0),
               None if zeros is None else _half8(zeros, 0.0))
        out = _launch([g], [g.shape[1]], mul, [mat], layout, K, group_size, dtype)
    return out.view(*dC.shape[:-1], K)


def _marlin_shape(words: torch.Tensor, scales: torch.Tensor, group_size: int, name: str) -> int:
    if words.dim() != 2:
        raise ValueError(f"{name} must be [K/8, N], got shape {tuple(words.shape)}")
    K = words.shape[0] * kernels.FP4_PER_UINT
    kernels._check_groups("scales", scales, K, words.shape[1], group_size)
    return K


def marlin_gemm_fp4_backward(dC: torch.Tensor, B_packed: torch.Tensor, scales: torch.Tensor,
                             group_size: int = 32,
                             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dA = dC @ dequant(B_packed, scales)^T, the input gradient of marlin_gemm_fp4
    (kernels_core.py:1830-1937 has the forward): dC [*, N] -> [*, K], B_packed [K/8, N],
    scales [K/group_size, N]."""
    _lib.require_device(dC, B_packed, scales)
    K = _marlin_shape(B_packed, scales, group_size, "B_packed")
    return _linear(dC, B_packed, scales, None, 0, K, group_size, out_dtype)


def marlin_gemm_int4_backward(dC: torch.Tensor, B_packed: torch.Tensor, scales: torch.Tensor,
                              zeros: torch.Tensor, group_size: int = 32,
                              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dA = dC @ ((q - zeros) * scales)^T, the input gradient of marlin_gemm_int4
    (kernels_core.py:1959-2066 has the forward)."""
    _lib.require_device(dC, B_packed, scales, zeros)
    K = _marlin_shape(B_packed, scales, group_size, "B_packed")
    kernels._check_groups("zeros", zeros, K, B_packed.shape[1], group_size)
    return _linear(dC, B_packed, scales, zeros, 0, K, group_size, out_dtype)


def mmfp4_gemm_rowpacked_backward(dC: torch.Tensor, B_rows: torch.Tensor, scales: torch.Tensor,
                                  group_size: int = 128,
                                  out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dA = dC @ dequant(B_rows), the input gradient of mmfp4_gemm_rowpacked and MMFP4Linear
    (layers/mmfp4_linear.py:549-598): B_rows [N, K/8] words, read in place (K % 32 != 0: on a
    transposed copy), scales [K/group_size, N] or [N, K/group_size]."""
    _lib.require_device(dC, B_rows, scales)
    if B_rows.dim() != 2 or scales.dim() != 2:
        raise ValueError(f"B_rows must be [N, K/8] and scales rank-2, got {tuple(B_rows.shape)} "
                         f"and {tuple(scales.shape)}")
    N, K = B_rows.shape[0], B_rows.shape[1] * kernels.FP4_PER_UINT
    if group_size <= 0 or K % group_size != 0:
        raise ValueError(f"K={K} must be divisible by group_size={group_size}")
    if kernels._scales_layout(scales, N, K // group_size) == 1:
        scales = scales.t()
    if K % 32 != 0:
        return _linear(dC, kernels._packed(B_rows.t()), scales, None, 0, K, group_size, out_dtype)
    return _linear(dC, B_rows, scales, None, 1, K, group_size, out_dtype)


def mmfp4_fused_qkv_backward(dQ: torch.Tensor, dK: torch.Tensor, dV: torch.Tensor,
                             Q_packed: torch.Tensor, Q_scales: torch.Tensor,
                             K_packed: torch.Tensor, K_scales: torch.Tensor,
                             V_packed: torch.Tensor, V_scales: torch.Tensor,
                             group_size: int = 128,
                             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """The input gradient of mmfp4_fused_qkv (kernels_core.py:4875-4948 has the forward):
    dA = dQ @ Wq^T + dK @ Wk^T + dV @ Wv^T in one product over the three matrices' columns,
    the sum rounded once."""
    dev = _lib.require_device(dQ, dK, dV, Q_packed, Q_scales, K_packed, K_scales, V_packed,
                              V_scales)
    if out_dtype in (None, dQ.dtype):
        out = _lib.fast("qkv_backward", dQ, (dQ, dK, dV), (Q_packed, K_packed, V_packed),
                        (Q_scales, K_scales, V_scales), group_size)
        if out is not None:
            return out
    grads, mats, widths = [], [], []
    Kdim = Q_packed.shape[0] * kernels.FP4_PER_UINT
    dtype = out_dtype or dQ.dtype
    _type("out_dtype", dtype)
    with on_device(dev):
        for name, d, w, s in (("Q", dQ, Q_packed, Q_scales), ("K", dK, K_packed, K_scales),
                              ("V", dV, V_packed, V_scales)):
            if _marlin_shape(w, s, group_size, f"{name}_packed") != Kdim:
                raise ValueError(f"{name}_packed: K={w.shape[0] * 8} does not match K={Kdim}")
            if d.dtype != dQ.dtype or d.shape[:-1] != dQ.shape[:-1]:
                raise ValueError(f"d{name} {d.dtype} {tuple(d.shape)} does not match dQ "
                                 f"{dQ.dtype} {tuple(dQ.shape)}")
            grads.append(_flat(d, w.shape[1], f"d{name}"))
            widths.append(grads[-1].shape[1])
            mats.append((_words8(w), _half8(s, 1.0), None))
        mul = None
        if dQ.dtype != torch.float16:
            # one power of two per row for all three
            M, n = grads[0].shape[0], sum(widths)
            whole = torch.empty((M, n), dtype=torch.float16, device=dev)
            mul = torch.empty(M, dtype=torch.float32, device=dev)
            _lib.call("mm_grad_rows_multi",
                      (ctypes.c_void_p * 3)(*[g.data_ptr() for g in grads]), _TYPES[dQ.dtype], 3,
                      (ctypes.c_int * 3)(*widths), _lib.ptr(whole), _lib.ptr(mul), M,
                      _lib.stream_of(whole))
            grads = list(whole.split(widths, 1))
            widths = [n] * 3
        out = _launch(grads, widths, mul, mats, 0, Kdim, group_size, dtype)
    return out.view(*dQ.shape[:-1], Kdim)


def _check_pair(x_k: int | None, gate_packed, gate_scales, up_packed, up_scales, group_size: int,
                row_packed: bool) -> tuple[int, int]:
    if gate_packed.dim() != 2 or tuple(up_packed.shape) != tuple(gate_packed.shape):
        raise ValueError(f"up_packed must match gate_packed shape {tuple(gate_packed.shape)}, "
                         f"got {tuple(up_packed.shape)}")
    d0, d1 = gate_packed.shape
    N, K = (d0, 8 * d1) if row_packed else (d1, 8 * d0)
    if x_k is not None and x_k != K:
        raise ValueError(f"K mismatch: x has K={x_k}, but packed tensors imply K={K}")
    kernels._check_groups("gate_scales", gate_scales, K, N, group_size)
    kernels._check_groups("up_scales", up_scales, K, N, group_size)
    return N, K


def fused_gate_up_swiglu(x: torch.Tensor, gate_packed: torch.Tensor, gate_scales: torch.Tensor,
                         up_packed: torch.Tensor, up_scales: torch.Tensor, group_size: int = 128,
                         row_packed: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """The gated feed-forward block of mmfp4_fused_gate_up[_marlin] for training: returns
    h = silu(x @ Wg) * (x @ Wu) [*, N] and gate_up = [x @ Wg | x @ Wu] [*, 2N], which
    fused_gate_up_swiglu_backward starts from; both fp16, rounded from the same fp32 sums in
    one launch.  Marlin words [K/8, N], or with row_packed [N, K/8]; scales [K/group_size, N].
    Shapes that the one-launch kernels do not take (N % 8 != 0; above 32 rows K % 64 != 0;
    row-packed words whose group size is no multiple of 32, or 64 above 32 rows) run two
    products, and SiLU then sees the fp16 ones.  Where x requires a gradient, h is
    differentiable in x, and gate_up is not."""
    if kernels._wants_grad(x):
        from .autograd import GateUp
        return GateUp.apply(x, gate_packed, gate_scales, up_packed, up_scales, group_size,
                            row_packed, False)
    dev = _lib.require_device(x, gate_packed, gate_scales, up_packed, up_scales)
    if x.dim() == 0 or not x.is_floating_point():
        raise ValueError(f"x must be a floating tensor [*, K], got {x.dtype} {tuple(x.shape)}")
    out = _lib.fast("gate_up_keep", x, x, gate_packed, gate_scales, up_packed, up_scales,
                    group_size, row_packed)
    if out is not None:
        return out
    N, K = _check_pair(x.shape[-1], gate_packed, gate_scales, up_packed, up_scales, group_size,
                       row_packed)
    lead = x.shape[:-1]
    with on_device(dev):
        a = plain(kernels._half(x.reshape(-1, K)))
        M = a.shape[0]
        one_launch = kernels.rowpacked_gemm_supported(max(M, 1), N, K, group_size) \
            if row_packed else M <= 32 or K % 64 == 0
        if N % 8 != 0 or not one_launch:
            if row_packed:
                gate_packed, up_packed = (kernels._packed(w.t()) for w in
                                          (gate_packed, up_packed))
            g, u = (kernels.marlin_gemm_fp4(a, w, s, group_size).reshape(*lead, N) for w, s in
                    ((gate_packed, gate_scales), (up_packed, up_scales)))
            h = (torch.nn.functional.silu(g.float()) * u.float()).half()
            return h, torch.cat([g, u], -1)
        h = torch.empty((*lead, N), dtype=torch.float16, device=dev)
        gate_up = torch.empty((*lead, 2 * N), dtype=torch.float16, device=dev)
        if M > 0:
            stream = _lib.raw_stream(dev.index)
            ws = _lib.workspace_on(dev.index, stream, kernels._ws_bytes(M, 2 * N, K))
            ops = [plain(t) for t in (kernels._packed(gate_packed), kernels._half(gate_scales),
                                      kernels._packed(up_packed), kernels._half(up_scales))]
            _lib.call("mm_fp4_gate_up_keep", _lib.ptr(a), *map(_lib.ptr, ops), _lib.ptr(h),
                      _lib.ptr(gate_up), int(row_packed), M, N, K, group_size, _lib.ptr(ws),
                      ws.numel(), stream)
    return h, gate_up


def fused_gate_up_swiglu_backward(dh: torch.Tensor, gate_up: torch.Tensor,
                                  gate_packed: torch.Tensor, gate_scales: torch.Tensor,
                                  up_packed: torch.Tensor, up_scales: torch.Tensor,
                                  group_size: int = 128, row_packed: bool = False,
                                  out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """The input gradient of fused_gate_up_swiglu: dh [*, N], gate_up [*, 2N] as the forward
    returned it -> dx [*, K] = dg @ Wg^T + du @ Wu^T with
    dg = dh * u * sig(g) * (1 + g * (1 - sig(g))), du = dh * silu(g)."""
    dev = _lib.require_device(dh, gate_up, gate_packed, gate_scales, up_packed, up_scales)
    N, K = _check_pair(None, gate_packed, gate_scales, up_packed, up_scales, group_size,
                       row_packed)
    if out_dtype in (None, dh.dtype):
        out = _lib.fast("gate_up_backward", dh, dh, gate_up, gate_packed, gate_scales, up_packed,
                        up_scales, group_size, row_packed)
        if out is not None:
            return out
    if tuple(gate_up.shape) != (*dh.shape[:-1], 2 * N):
        raise ValueError(f"gate_up shape {tuple(gate_up.shape)} != "
                         f"{(*dh.shape[:-1], 2 * N)}")
    if gate_up.dtype != torch.float16:
        raise TypeError(f"gate_up must be fp16, as the forward returns it, got {gate_up.dtype}")
    dtype = out_dtype or dh.dtype
    _type("out_dtype", dtype)
    with on_device(dev):
        d = _flat(dh, N, "dh")
        M, N8 = d.shape
        gu = gate_up.reshape(M, 2 * N)
        if N8 != N:
            gu = torch.cat([_pad_to(t, N8) for t in gu.split(N, 1)], 1)
        gu = plain(gu)
        dgu = torch.empty((M, 2 * N8), dtype=torch.float16, device=dev)
        mul = torch.empty(M, dtype=torch.float32, device=dev)
        _lib.call("mm_swiglu_grad", _lib.ptr(d), _TYPES[d.dtype], _lib.ptr(gu), _lib.ptr(dgu),
                  _lib.ptr(mul), M, N8, _lib.stream_of(d))
        layout = int(row_packed)
        if row_packed and K % 32 != 0:
            gate_packed, up_packed = (kernels._packed(w.t()) for w in (gate_packed, up_packed))
            layout = 0
        mats = [(_words8(w, 1 - layout), _half8(s, 1.0), None)
                for w, s in ((gate_packed, gate_scales), (up_packed, up_scales))]
        out = _launch([dgu[:, :N8], dgu[:, N8:]], [2 * N8] * 2, mul, mats, layout, K, group_size,
                      dtype)
    return out.view(*dh.shape[:-1], K)
