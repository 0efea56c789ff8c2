"""Adapters of fp32 tokens: gradients far below what fp16 holds, and far above, come through as
they do through the layer beside them."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


class Case:
    def __init__(self, T, K, N, r, L, seed=0):
        gen = torch.Generator().manual_seed(seed + T + N)
        rnd = lambda *s, std=1.0: (torch.randn(s, generator=gen) * std).half().float().to(DEV)  # noqa
        self.T, self.K, self.N, self.r, self.L = T, K, N, r, L
        self.x, self.dy = rnd(T, K), torch.randn((T, N), generator=gen).to(DEV)
        self.a, self.b = rnd(L, r, K, std=K ** -0.5), rnd(L, N, r, std=0.05)
        self.ids = torch.randint(-1, L, (T,), generator=gen).to(DEV)
        self.s = 0.5 + torch.rand(L, generator=gen).to(DEV)
        self.dx_base = torch.randn((T, K), generator=gen).to(DEV)

    def check(self, got, with_base=True, extra=0.0):
        """dy in 11 bits but for what lies 2^-40 below a token's largest; H and dH in 22 bits of
        a token's or a tile's largest; fp32 sums and results.  extra: what dx_base is off by."""
        dx, da, db = got
        x, dy, a, b = (t.double() for t in (self.x, self.dy, self.a, self.b))
        ref = self.dx_base.double() if with_base else torch.zeros_like(x)
        tdx, one = ref.abs(), 2.0 ** -24
        da0, db0 = torch.zeros_like(a), torch.zeros_like(b)
        tda, tdb, lda, ldb = (torch.zeros_like(t) for t in (a, b, a, b))
        for e in range(self.L):
            k = self.ids == e
            s = self.s[e].double()
            h, dh = s * (x[k] @ a[e].t()), s * (dy[k] @ b[e])
            th, tdh = s * (x[k].abs() @ a[e].abs().t()), s * (dy[k].abs() @ b[e].abs())
            ref[k] += dh @ a[e]
            tdx[k] += tdh @ a[e].abs()
            da0[e], db0[e] = dh.t() @ x[k], dy[k].t() @ h
            tda[e], tdb[e] = tdh.t() @ x[k].abs(), dy[k].abs().t() @ th
            if k.any():
                # a tile's small tokens beside its largest: 2^-38 of that
                top = dy[k].abs().amax(1)
                lda[e] = 2.0 ** -37 * tdh.amax() * x[k].abs().sum(0)
                ldb[e] = 2.0 ** -37 * (th.amax(1) * top).amax() * (dy[k].abs() /
                                                                  top.unsqueeze(1)).sum(0)[:, None]
        n = (self.N + self.r + self.T) * 2 * one
        low = 2.0 ** -40 * self.N
        for name, g, r, t, l in (("dx", dx, ref, tdx, extra), ("da", da, da0, tda, lda),
                                 ("db", db, db0, tdb, ldb)):
            assert g.dtype == F32
            tol = one * r.abs() + (2.0 ** -11 + low + 2.0 ** -20 + n) * t + l + 2.0 ** -149
            assert ((g.double() - r).abs() <= tol).all(), name


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e-7, 1.0, 1e9, 1e30])
@pytest.mark.parametrize("T,K,N,r,L", [(3, 64, 40, 4, 2), (70, 100, 37, 8, 3),
                                       (900, 256, 136, 20, 2), (2500, 128, 72, 100, 1),
                                       (300, 64, 1, 1, 1)])
def test_sizes(T, K, N, r, L, size):
    c = Case(T, K, N, r, L)
    announce(f"fp32 adapters {T} {K} {N} {r} {L} {size}")
    c.dy *= size
    c.dx_base *= size
    c.check(mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s, dx_base=c.dx_base))
    c.check(mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s), with_base=False)


def test_tokens_of_different_sizes():
    """From 1e-20 to 1e20 in one batch: each token's dx is right for its own size."""
    c = Case(1000, 128, 72, 8, 3)
    c.dy *= (10.0 ** torch.linspace(-20, 20, 1000, device=DEV)).unsqueeze(1)[
        torch.randperm(1000, device=DEV)]
    c.dx_base.zero_()
    c.check(mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s, dx_base=c.dx_base))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_wide_gradients_of_fp16_tokens(dtype):
    """dx has the tokens' type; a token whose dy lies below fp16 still counts in da and db."""
    c = Case(200, 64, 48, 8, 2)
    c.dy = (c.dy * 1e-9).to(dtype)
    dx, da, db = mmfp4.lora_backward(c.dy, c.x.half(), c.a, c.b, c.ids, c.s)
    assert dx.dtype == F16
    want = mmfp4.lora_backward(c.dy.float(), c.x, c.a, c.b, c.ids, c.s)
    assert torch.equal(dx, want[0].half())
    assert torch.equal(da, want[1]) and torch.equal(db, want[2]) and da.any() and db.any()


def test_a_layer_trained_in_fp32():
    """The mean of a loss over many values, without a loss scale: gradients of 1e-9."""
    gen = torch.Generator().manual_seed(5)
    K, N, g, T = 256, 128, 64, 300
    w = (torch.randn((N, K), generator=gen) * 0.05).half().to(DEV)
    words, scales = mmfp4.quantize_fp4(w, group_size=g)
    W = mmfp4.dequant_fp4(words, scales, K, N, g).double()
    m = mmfp4.LoRALinear(mmfp4.MarlinLinear(words, scales, None, g), 8, 2, dtype=F32)
    c = Case(T, K, N, 8, 2)
    with torch.no_grad():
        m.lora_a.copy_(c.a)
        m.lora_b.copy_(c.b)
    x = c.x.clone().requires_grad_(True)
    y = m(x, c.ids)
    assert y.dtype == F32
    got = torch.autograd.grad(y, (x, m.lora_a, m.lora_b), c.dy * 1e-9)
    c.dy, c.s = c.dy * 1e-9, torch.ones(2, device=DEV)
    c.dx_base = c.dy.double() @ W.t()
    # the layer's own gradient: dy in 11 bits, fp32 sums
    c.check(got, extra=(2.0 ** -11 + 2 * N * 2.0 ** -24) * (c.dy.double().abs() @ W.abs().t()))


def test_captured():
    c = Case(300, 64, 48, 8, 3)

    def step():
        return mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s, dx_base=c.dx_base)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    gen = torch.Generator().manual_seed(6)
    for i in range(4):
        for t in (c.x, c.dy, c.dx_base):
            t.copy_(torch.randn(t.shape, generator=gen) * 10.0 ** -(4 * i))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(held, step()):
            assert torch.equal(p, q), i
