"""The products as nodes: a result whose activations require a gradient carries one, so that
lora_add beside it sends the whole gradient back."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from mmfp4.layers.mmfp4_linear import mmfp4_gemm as rows_gemm

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


class Weights:
    def __init__(self, seed, N, K, g):
        self.gen = torch.Generator().manual_seed(seed)
        w = (torch.randn((N, K), generator=self.gen) * 0.05).half().to(DEV)
        self.N, self.K, self.g = N, K, g
        self.w, self.s = mmfp4.quantize_fp4(w, group_size=g)
        self.w4, self.s4, self.z4 = mmfp4.pack_u4_weights(w, group_size=g)
        self.rows, self.st = self.w.t().contiguous(), self.s.t().contiguous()
        self.W = mmfp4.dequant_fp4(self.w, self.s, K, N, g).t().double()
        self.W4 = mmfp4.dequant_int4(self.w4, self.s4, self.z4, K, N, g).t().double()

    def randn(self, *shape, dtype=F16):
        return torch.randn(shape, generator=self.gen).to(DEV, dtype)

    def calls(self):
        """Name, forward, its matrix [N, K]."""
        w, s, g = self.w, self.s, self.g
        yield "fp4", lambda x: mmfp4.marlin_gemm_fp4(x, w, s, g), self.W
        yield "u4", lambda x: mmfp4.marlin_gemm_int4(x, self.w4, self.s4, self.z4, g), self.W4
        yield "gemv", lambda x: mmfp4.decode_gemv_fp4(x, w, s, g), self.W
        yield "op", lambda x: mmfp4.GemmFp4()(x, w, s, g), self.W
        yield "mmfp4", lambda x: mmfp4.mmfp4_gemm(x, w, s, g), self.W
        yield "mmfp4 transposed", lambda x: mmfp4.mmfp4_gemm(x, w, self.st, g), self.W
        yield "rows", lambda x: rows_gemm(x, self.rows, s, g), self.W
        if self.N % 8 == 0:
            yield "in place", lambda x: mmfp4.mmfp4_gemm_rowpacked(x, self.rows, s, g), self.W


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,N", [(1, 96), (9, 101), (70, 96)])
def test_products(M, N, dtype):
    o = Weights(1, N, 256, 64)
    for name, f, W in o.calls():
        x = o.randn(M, o.K, dtype=dtype)
        still = f(x)
        assert not still.requires_grad
        x.requires_grad_(True)
        with torch.no_grad():
            assert not f(x).requires_grad
        y = f(x)
        assert y.dtype == F16 and torch.equal(y.detach(), still), name
        dy = o.randn(M, N)
        dx, = torch.autograd.grad(y, x, dy)
        assert dx.dtype == dtype and dx.shape == x.shape
        ref, terms = dy.double() @ W, dy.double().abs() @ W.abs()
        # half a step of the result, and fp32 sums of N terms
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + (N + 2) * 2.0 ** -24 * terms + 2.0 ** -25
        assert ((dx.double() - ref).abs() <= tol).all(), name
        dx2, = torch.autograd.grad(f(x).mul_(2), x, dy)     # changed in place
        # doubling commutes with rounding but below the normal fp16 numbers, where steps are
        # 2^-24: |round(2v) - 2 round(v)| <= 2^-25 + 2 * 2^-25 < 2^-23
        assert ((dx2.double() - 2 * dx.double()).abs() <= 2.0 ** -23).all(), name


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", [(256,), (5, 256), (2, 30, 256)])
@pytest.mark.parametrize("N", [64, 41])
def test_fused_qkv(shape, N, dtype):
    o, kv = Weights(2, N, 256, 64), Weights(3, 32, 256, 64)
    mats = (o.w, o.s, kv.w, kv.s, kv.w, kv.s)
    x = o.randn(*shape, dtype=dtype)
    still = mmfp4.mmfp4_fused_qkv(x, *mats, o.g)
    x.requires_grad_(True)
    out = mmfp4.mmfp4_fused_qkv(x, *mats, o.g)
    assert all(torch.equal(a.detach(), b) for a, b in zip(out, still))
    d = [o.randn(*t.shape) for t in out]
    dx, = torch.autograd.grad(out, x, d)
    want = mmfp4.mmfp4_fused_qkv_backward(*d, *mats, o.g, out_dtype=dtype)
    assert dx.dtype == dtype and torch.equal(dx, want.view(shape))
    q, k, v = mmfp4.mmfp4_fused_qkv(x, *mats, o.g)
    dx, = torch.autograd.grad(k.mul_(1), x, d[1])           # one of the three
    zero = [torch.zeros_like(d[0]), d[1], torch.zeros_like(d[2])]
    want = mmfp4.mmfp4_fused_qkv_backward(*zero, *mats, o.g, out_dtype=dtype)
    assert torch.equal(dx, want.view(shape))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,K", [(20, 256), (40, 288)])      # one launch, two products
def test_gate_up_that_keeps(M, K, dtype):
    o = Weights(4, 96, K, 32)
    x = o.randn(M, K, dtype=dtype)
    mats = (o.w, o.s) * 2
    h0, kept0 = mmfp4.fused_gate_up_swiglu(x, *mats, o.g)
    x.requires_grad_(True)
    h, kept = mmfp4.fused_gate_up_swiglu(x, *mats, o.g)
    assert h.requires_grad and not kept.requires_grad and h.dtype == F16
    assert torch.equal(h.detach(), h0) and torch.equal(kept, kept0)
    dh = o.randn(*h.shape)
    dx, = torch.autograd.grad(h, x, dh)
    assert torch.equal(dx, mmfp4.fused_gate_up_swiglu_backward(dh, kept, *mats, o.g,
                                                               out_dtype=dtype))


def test_adapters_beside_a_product():
    """The whole gradient reaches x: through the base and through the adapter."""
    o = Weights(5, 64, 256, 64)
    r = 4
    a, b = o.randn(r, o.K), o.randn(o.N, r)
    for name, f, W in o.calls():
        x = o.randn(30, o.K).requires_grad_(True)
        y = mmfp4.lora_add(f(x), x, a, b, scaling=0.25)
        dy = o.randn(30, o.N)
        dx, = torch.autograd.grad(y, x, dy)
        full = W + 0.25 * b.double() @ a.double()
        ref = dy.double() @ full
        terms = dy.double().abs() @ (W.abs() + 0.25 * b.double().abs() @ a.double().abs())
        # two gradients and their sum, a rounding of half a step (2^-11) each
        assert ((dx.double() - ref).abs() <= 3 * 2.0 ** -11 * terms).all(), name


def test_step_captured():
    o = Weights(6, 128, 256, 64)
    x = o.randn(40, o.K).requires_grad_(True)

    def step():
        q, k, v = mmfp4.mmfp4_fused_qkv(x, *(o.w, o.s) * 3, o.g)
        y = q + k * v + mmfp4.marlin_gemm_fp4(x, o.w, o.s, o.g)
        return torch.autograd.grad(y.float().square().sum(), x)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        with torch.no_grad():
            x.copy_(o.randn(40, o.K))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], step()[0])


def test_out_takes_no_part():
    o = Weights(7, 64, 256, 64)
    x = o.randn(3, 256).requires_grad_(True)
    out = torch.empty((3, 64), dtype=F16, device=DEV)
    assert mmfp4.dispatch_gemm_fp4(None, x, o.w, o.s, 3, 64, 256, o.g, out=out) is out
    assert not out.requires_grad
    assert mmfp4.dispatch_gemm_fp4(None, x, o.w, o.s, 3, 64, 256, o.g).requires_grad
