"""Biases of the quantized layers that are trained: beside adapters, and under capture."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from mmfp4.layers import MMFP4Linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def layers(gen, K, N, g, dtype):
    w = (torch.randn((N, K), generator=gen) * 0.05).half().to(DEV)
    words, scales = mmfp4.quantize_fp4(w, group_size=g)
    bias = lambda: torch.randn(N, generator=gen).to(DEV, dtype)            # noqa: E731
    q = mmfp4.QuantizedTensor(words, scales, "fp4", g, (N, K))
    yield "quantized", mmfp4.QuantizedLinear(q, bias())
    yield "marlin", mmfp4.MarlinLinear(words, scales, bias(), g)
    yield "rows", MMFP4Linear(words.t().contiguous(), scales, bias(), g)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T", [5, 100, 300])
def test_beside_adapters(T, dtype):
    gen = torch.Generator().manual_seed(1)
    K, N, g = 256, 96, 64
    for name, layer in layers(gen, K, N, g, dtype):
        m = mmfp4.LoRALinear(layer, rank=8, num_adapters=2,
                             dtype=F16 if dtype == F32 else dtype)
        with torch.no_grad():
            m.lora_b.copy_(torch.randn(m.lora_b.shape, generator=gen) * 0.05)
        ids = torch.randint(-1, 2, (T,), generator=gen).to(DEV)
        x = torch.randn((T, K), generator=gen).to(DEV, dtype).requires_grad_(True)
        dy = torch.randn((T, N), generator=gen).to(DEV, dtype)
        y = m(x, ids)
        frozen = torch.autograd.grad(y, (x, m.lora_a, m.lora_b), dy)
        layer.bias.requires_grad_(True)
        z = m(x, ids)
        db, dx, da, dlb = torch.autograd.grad(z, (layer.bias, x, m.lora_a, m.lora_b), dy)
        # fp32 sums of T gradients, rounded once to the bias's type
        ref, terms = dy.double().sum(0), dy.double().abs().sum(0)
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + T * 2.0 ** -24 * terms + 2.0 ** -25
        assert ((db.double() - ref).abs() <= tol).all(), name
        for got, want in ((z, y), (dx, frozen[0]), (da, frozen[1]), (dlb, frozen[2])):
            assert torch.equal(got, want), name
        only, = torch.autograd.grad(m(x.detach(), ids), layer.bias, dy)
        assert torch.equal(only, db), name
        m.requires_grad_(False)                      # the bias alone
        layer.bias.requires_grad_(True)
        only, = torch.autograd.grad(m(x.detach(), ids), layer.bias, dy)
        assert torch.equal(only, db), name


def test_beside_adapters_captured():
    """Replayed several times on new inputs, against eager steps."""
    gen = torch.Generator().manual_seed(2)
    T, K, N, g = 5000, 128, 64, 64
    layer = next(layers(gen, K, N, g, F16))[1]
    layer.bias.requires_grad_(True)
    m = mmfp4.LoRALinear(layer, rank=4)
    x = torch.randn((T, K), generator=gen).to(DEV, F16)
    dy = torch.randn((T, N), generator=gen).to(DEV, F16)

    def step():
        return torch.autograd.grad(m(x), (layer.bias, m.lora_a, m.lora_b), dy)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=gen))
        dy.copy_(torch.randn(dy.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("wants", [False, True])
def test_capture_beside_a_living_graph_is_refused(wants):
    """An eager graph of the bias is alive on another stream: the captured forward pass raises
    (a backward pass would end the process)."""
    gen = torch.Generator().manual_seed(3)
    for name, layer in layers(gen, 64, 64, 64, F16):
        layer.bias.requires_grad_(True)
        x = torch.randn((4, 64), generator=gen).to(DEV, F16)
        alive = layer(x)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            y = x.clone().requires_grad_(wants)
            for f in (layer, mmfp4.LoRALinear(layer, 4)):
                with pytest.raises(RuntimeError, match="another stream"):
                    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                        f(y)
                with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                    f(y)                             # nothing to go back through
        torch.cuda.synchronize()
        assert alive.isfinite().all()
