"""Autograd through the quantized layers and their adapters: the gradients are those of the
explicit backward calls (which are tested against the formulas), and a training step of a block
made of them runs, also captured."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from mmfp4.layers import MMFP4Linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def weight(gen, n, k):
    return (torch.randn((n, k), generator=gen) * 0.05).half().to(DEV)


def layers(gen, K, N, g):
    """One of each kind, with a bias, and its dequantized weight [N, K]."""
    w = weight(gen, N, K)
    words, scales = mmfp4.quantize_fp4(w, group_size=g)
    bias = torch.randn(N, generator=gen).half().to(DEV)
    W = mmfp4.dequant_fp4(words, scales, K, N, g).t().double()
    q = mmfp4.QuantizedTensor(words, scales, "fp4", g, (N, K))
    yield "quantized", mmfp4.QuantizedLinear(q, bias), W
    yield "marlin", mmfp4.MarlinLinear(words, scales, bias, g), W
    yield "rows", MMFP4Linear(words.t().contiguous(), scales, bias, g), W
    rot = torch.linalg.qr(torch.randn((K, K), generator=gen))[0].half().to(DEV)
    yield "rotated", mmfp4.QuantizedLinear(mmfp4.QuantizedTensor(
        words, scales, "fp4", g, (N, K), True, rot), bias), W @ rot.double().t()
    w4, s4, z4 = mmfp4.pack_u4_weights(w, group_size=g)
    W4 = mmfp4.dequant_int4(w4, s4, z4, K, N, g).t().double()
    yield "int4", mmfp4.QuantizedLinear(mmfp4.QuantizedTensor(w4, s4, "int4", g, (N, K),
                                                              zeros=z4), bias), W4


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("shape", [(3,), (2, 40)])
def test_layers(shape, dtype):
    gen = torch.Generator().manual_seed(1)
    for name, layer, W in layers(gen, 256, 96, 64):
        x = torch.randn((*shape, 256), generator=gen).to(DEV, dtype)
        with torch.no_grad():
            still = layer(x)
        assert not still.requires_grad and still.dtype == dtype
        x.requires_grad_(True)
        y = layer(x)
        assert torch.equal(y.detach(), still), name
        dy = torch.randn(y.shape, generator=gen).to(DEV, dtype)
        dx, = torch.autograd.grad(y, x, dy)
        assert dx.dtype == dtype and dx.shape == x.shape
        ref = dy.double() @ W
        # half a step of the result; fp32 is carried in fp16 (2^-11 of every term); the rotation
        # is a product in fp32
        terms = dy.double().abs() @ W.abs()
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -11 * terms
        if name == "rotated":
            tol = tol + 2.0 ** -10 * terms.max()
        assert ((dx.double() - ref).abs() <= tol).all(), name


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gate_up(dtype, rows):
    gen = torch.Generator().manual_seed(2)
    K, N, g = 256, 128, 64
    mats = []
    for _ in range(2):
        words, scales = mmfp4.quantize_fp4(weight(gen, N, K), group_size=g)
        mats += [words.t().contiguous() if rows else words, scales]
    x = torch.randn((2, 30, K), generator=gen).to(DEV, dtype).requires_grad_(True)
    h = mmfp4.gate_up_swiglu(x, *mats, g, rows)
    dh = torch.randn(h.shape, generator=gen).to(DEV, dtype)
    dx, = torch.autograd.grad(h, x, dh)
    kept, gu = mmfp4.fused_gate_up_swiglu(x.detach(), *mats, g, rows)
    assert h.dtype == dtype and torch.equal(h, kept.to(dtype))
    assert torch.equal(dx, mmfp4.fused_gate_up_swiglu_backward(dh, gu, *mats, g, rows))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N", [128, 36])
def test_results_may_be_changed_in_place(N, dtype):
    gen = torch.Generator().manual_seed(12)
    K, g = 64, 64
    w, s = mmfp4.quantize_fp4(weight(gen, N, K), group_size=g)
    lib = mmfp4.get_default_library()
    w4, s4, z4 = mmfp4.pack_u4_weights(weight(gen, N, K), group_size=g)
    for shape in ((K,), (3, K), (2, 20, K)):
        x = torch.randn(shape, generator=gen).to(DEV, dtype).requires_grad_(True)
        calls = [lambda: mmfp4.quantized_linear(x, w, s, g),
                 lambda: lib.fp4_gemm(x, w, s, N, K, g),
                 lambda: lib.int4_gemm(x, w4, s4, N, K, g, z4),
                 lambda: mmfp4.gate_up_swiglu(x, w, s, w, s, g)]
        for f in calls if len(shape) > 1 else calls[-1:]:
            y = f()
            dx, = torch.autograd.grad(y, x, torch.ones_like(y))
            dx2, = torch.autograd.grad(f().mul_(2), x, torch.ones_like(y))
            assert dx.shape == x.shape and torch.equal(dx2, 2 * dx)


@pytest.mark.parametrize("T", [5, 300])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_adapters(dtype, T):
    gen = torch.Generator().manual_seed(3)
    K, N, g = 256, 96, 64
    ids = torch.randint(-1, 3, (T,), generator=gen).to(DEV)
    for name, layer, _ in layers(gen, K, N, g):
        m = mmfp4.LoRALinear(layer, rank=8, num_adapters=3, dtype=dtype,
                             scaling=torch.tensor([0.5, 1.0, 2.0]))
        x = torch.randn((T, K), generator=gen).to(DEV, dtype)
        assert torch.equal(m(x, ids).detach(), layer(x))       # lora_b is zeros
        with torch.no_grad():
            m.lora_b.copy_(torch.randn(m.lora_b.shape, generator=gen))
        x.requires_grad_(True)
        y = m(x, ids)
        base = layer(x.detach()).detach()
        assert torch.equal(y.detach(), mmfp4.lora_add(base, x.detach(), m.lora_a.detach(),
                                                      m.lora_b.detach(), ids, m.scaling))
        dy = torch.randn(y.shape, generator=gen).to(DEV, dtype)
        got = torch.autograd.grad(y, (x, m.lora_a, m.lora_b), dy)
        want = mmfp4.lora_backward(dy, x.detach(), m.lora_a.detach(), m.lora_b.detach(), ids,
                                   m.scaling, dx_base=layer.input_grad(dy))
        for a, b in zip(got, want):
            assert a.dtype == b.dtype and torch.equal(a, b), name
        with torch.no_grad():
            assert torch.equal(m(x, ids), y)


@pytest.mark.parametrize("K,N,g", [(72, 35, 24), (264, 100, 8), (64, 4, 64)])
@pytest.mark.parametrize("M", [1, 50])
def test_odd_layers(M, K, N, g):
    """Widths that the kernels take on padded or transposed copies."""
    gen = torch.Generator().manual_seed(10)
    for name, layer, W in layers(gen, K, N, g):
        x = torch.randn((M, K), generator=gen).to(DEV, F16).requires_grad_(True)
        layer(x).mul_(2)                                       # results may be changed in place
        m = mmfp4.LoRALinear(layer, rank=3)
        dy = torch.randn((M, N), generator=gen).to(DEV, F16)
        ref, terms = dy.double() @ W, dy.double().abs() @ W.abs()
        tol = 2.0 ** -11 * ref.abs() + 2.0 ** -11 * terms      # as in test_layers
        if name == "rotated":
            tol = tol + 2.0 ** -10 * terms.max()
        for f in (layer, m):                                   # lora_b is zeros
            dx, = torch.autograd.grad(f(x), x, dy)
            # LoRALinear rounds the sum of two gradients once more
            assert ((dx.double() - ref).abs() <= 2 * tol).all(), (name, f)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_bias_gets_its_gradient(dtype):
    gen = torch.Generator().manual_seed(9)
    for name, layer, _ in layers(gen, 256, 96, 64):
        if isinstance(layer, mmfp4.QuantizedLinear) or name == "marlin":
            layer.bias = layer.bias.to(dtype)
        layer.bias.requires_grad_(True)
        x = torch.randn((5, 256), generator=gen).to(DEV, dtype)
        dy = torch.randn((5, 96), generator=gen).to(DEV, dtype)
        for wants in (False, True):
            x.requires_grad_(wants)
            db, = torch.autograd.grad(layer(x), layer.bias, dy)
            # five terms, each sum rounded to the type
            tol = 5 * torch.finfo(dtype).eps * dy.double().abs().sum(0) + 1e-6
            assert ((db.double() - dy.double().sum(0)).abs() <= tol).all(), (name, wants)


def test_twice_is_refused():
    """A gradient of a gradient is an error, not a silent zero."""
    gen = torch.Generator().manual_seed(6)
    x = torch.randn((4, 256), generator=gen).to(DEV, F16).requires_grad_(True)
    for name, layer, _ in layers(gen, 256, 96, 64):
        for f in (layer, mmfp4.LoRALinear(layer, rank=4)):
            dx, = torch.autograd.grad(f(x).square().sum(), x, create_graph=True)
            with pytest.raises(RuntimeError, match="once_differentiable"):
                dx.sum().backward()


def test_lora_add_as_a_node():
    """base, x and factors with gradients of their own, fp32 factors."""
    gen = torch.Generator().manual_seed(4)
    T, K, N = 40, 64, 48
    base, x = (torch.randn((T, n), generator=gen).to(DEV, F16).requires_grad_(True)
               for n in (N, K))
    a = torch.randn((4, K), generator=gen).to(DEV).requires_grad_(True)
    b = torch.randn((N, 4), generator=gen).to(DEV).requires_grad_(True)
    y = mmfp4.lora_add(base, x, a, b, scaling=0.5)
    dy = torch.randn((T, N), generator=gen).to(DEV, F16)
    gb, gx, ga, gbb = torch.autograd.grad(y, (base, x, a, b), dy)
    assert torch.equal(gb, dy)
    want = mmfp4.lora_backward(dy, x.detach(), a.detach(), b.detach(), scaling=0.5)
    assert torch.equal(gx, want[0]) and torch.equal(ga, want[1]) and torch.equal(gbb, want[2])
    assert ga.dtype == F32 and gbb.dtype == F32
    with pytest.raises(ValueError, match="out="):
        mmfp4.lora_add(base, x, a, b, out=torch.empty_like(dy))
    with pytest.raises(ValueError, match="scaling.detach"):
        mmfp4.lora_add(base, x, a, b, scaling=torch.ones(1, device=DEV, requires_grad=True))
    only = torch.autograd.grad(mmfp4.lora_add(base, x.detach(), a.detach(), b.detach()), base, dy)
    assert torch.equal(only[0], dy)


class Block(torch.nn.Module):
    """q/k/v-like projections with adapters, a gated feed-forward block, a residual."""

    def __init__(self, gen, dtype, H=128, I=192, g=64):
        super().__init__()
        q = [mmfp4.quantize_fp4(weight(gen, n, k), group_size=g)
             for n, k in ((H, H), (I, H), (I, H), (H, I))]
        lin = [mmfp4.MarlinLinear(w, s, None, g) for w, s in (q[0], q[3])]
        self.mix = mmfp4.LoRALinear(lin[0], 4, 2, 0.5, dtype)
        self.down = mmfp4.LoRALinear(lin[1], 4, 2, 0.5, dtype)
        self.pair, self.g = (*q[1], *q[2]), g

    def forward(self, x, ids):
        x = x + self.mix(x, ids)
        return x + self.down(mmfp4.gate_up_swiglu(x, *self.pair, self.g), ids)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_block_trains(dtype):
    """Steps run, the adapters in use get gradients and the others none, weights stay."""
    gen = torch.Generator().manual_seed(5)
    m = Block(gen, dtype)
    x = torch.randn((100, 128), generator=gen).to(DEV, dtype)
    ids = torch.zeros(100, dtype=torch.int32, device=DEV)
    words = m.pair[0].clone()
    opt = torch.optim.SGD(m.parameters(), lr=1e-2)
    for _ in range(3):
        opt.zero_grad()
        m(x, ids).float().square().mean().backward()
        for p in m.parameters():
            assert p.grad is not None and p.grad.isfinite().all() and not p.grad[1].any()
        opt.step()
    assert m.mix.lora_b[0].any() and not m.mix.lora_b[1].any()
    assert torch.equal(words, m.pair[0])


def test_block_captured():
    """Forward and backward of the block captured and replayed, against eager steps."""
    gen = torch.Generator().manual_seed(6)
    m = Block(gen, BF16)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(p.shape, generator=gen) * 0.1)
    x = torch.randn((100, 128), generator=gen).to(DEV, BF16)
    ids = torch.zeros(100, dtype=torch.int32, device=DEV)

    def grads():
        return torch.autograd.grad(m(x, ids).float().square().mean(), list(m.parameters()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        for _ in range(2):
            grads()
        with torch.cuda.graph(graph, stream=side):
            held = grads()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        x.copy_(torch.randn(x.shape, generator=gen))
        ids.copy_(torch.randint(-1, 2, (100,), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, grads()):
            assert torch.equal(a, b), i


def test_capture_beside_a_living_graph_is_refused():
    """An eager graph of the same leaves is alive on another stream: the forward pass raises
    under capture, before torch's engine meets it."""
    gen = torch.Generator().manual_seed(7)
    m = Block(gen, F16)
    x = torch.randn((40, 128), generator=gen).to(DEV, F16)
    alive = m(x, torch.zeros(40, dtype=torch.int32, device=DEV))
    ids = torch.zeros(40, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with pytest.raises(RuntimeError, match="another stream"):
            with torch.cuda.graph(graph, stream=side):
                m(x, ids)
    torch.cuda.synchronize()
    assert alive.isfinite().all()


def test_capture_behind_other_operations_is_refused():
    """The same where the leaf lies behind torch's own operations."""
    gen = torch.Generator().manual_seed(8)
    layer = next(iter(layers(gen, 64, 64, 64)))[1]
    p = torch.randn((5, 64), generator=gen).to(DEV, F16).requires_grad_(True)
    alive = p * 2
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with pytest.raises(RuntimeError, match="another stream"):
            with torch.cuda.graph(graph, stream=side):
                layer((p + 1).relu())
    torch.cuda.synchronize()
    assert alive.isfinite().all()
