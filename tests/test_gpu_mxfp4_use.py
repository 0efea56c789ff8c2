"""MXFP4 products, routing and experts as a program uses them together: captured into graphs and
replayed beside eager calls, on two streams at once, on a stream that is not the current one's
default, and as an experts' block behind its router, forward and backward."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import DEV, announce

pytestmark = pytest.mark.gpu


class Calls:
    """Every path: rows quantized by the product itself, streamed from codes, tiles of each size
    with K whole and split, K that is no multiple of 128; gradients with N split; both forms of
    the experts' block; routing and its gradient, few tokens and many."""

    def __init__(self, seed):
        gen = torch.Generator().manual_seed(seed)
        self.gen = gen
        rnd = lambda *s: torch.randn(s, generator=gen).to(DEV)              # noqa: E731
        self.wide = mmfp4.mxfp4_quantize(rnd(512, 2048) * 0.02)
        self.odd = mmfp4.mxfp4_quantize(rnd(72, 480) * 0.02)
        self.x = {m: rnd(m, 2048).bfloat16() for m in (1, 20, 48, 70, 300, 700)}
        self.xo = {m: rnd(m, 480).half() for m in (2, 90)}
        self.dy = {m: rnd(m, 512).to(t) for m, t in ((1, torch.float32), (50, torch.float16),
                                                     (300, torch.bfloat16))}
        self.gu = mmfp4.mxfp4_quantize(rnd(8, 2 * 160, 256) * 0.05)
        self.dn = mmfp4.mxfp4_quantize(rnd(8, 256, 160) * 0.05)
        self.h = {t: rnd(t, 256).half() for t in (3, 100)}
        self.gate, self.bias = rnd(256, 8) * 0.05, rnd(8) * 0.01
        self.logits = rnd(2100, 128)

    def inputs(self):
        return [*self.x.values(), *self.xo.values(), *self.dy.values(), *self.h.values(),
                self.logits]

    def renew(self):
        for x in self.inputs():
            x.copy_(torch.randn(x.shape, generator=self.gen))

    def step(self):
        out = [mmfp4.mxfp4_gemm(x, *self.wide) for x in self.x.values()]
        out += [mmfp4.mxfp4_gemm(x, *self.odd, torch.float32) for x in self.xo.values()]
        out += [mmfp4.mxfp4_gemm_backward(dy, *self.wide) for dy in self.dy.values()]
        for x in self.x.values():
            out += mmfp4.mxfp4_quantize(x)
        out.append(mmfp4.mxfp4_dequantize(*self.odd))
        for h in self.h.values():
            w, ids = mmfp4.moe_route(h.float() @ self.gate, 2, bias=self.bias, num_groups=2)
            out += [w, ids, mmfp4.moe_mlp_mxfp4(h, *self.gu, *self.dn, ids, w)]
        w, ids = mmfp4.moe_route(self.logits, 6, scoring="softmax")
        out += [w, ids, mmfp4.moe_route_backward(w, self.logits, ids, scoring="softmax")]
        return out


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("binding", [True, False])
def test_graphs_beside_eager_calls(binding, monkeypatch):
    if not binding:
        monkeypatch.setattr("mmfp4._lib._binding", False)
        monkeypatch.setattr("mmfp4.kernels._BINDING", False)
    sets = [Calls(s) for s in (1, 2)]
    for c in sets:
        c.step()
    torch.cuda.synchronize()
    mmfp4.release_workspaces()
    graphs, held = [], []
    for c in sets:
        announce("capture")
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(c.step())
    streams = [torch.cuda.Stream() for _ in sets]
    for order in ([1], [0], [0, 1], [1, 0], [0, 1]):
        for c in sets:
            c.renew()
        torch.cuda.synchronize()
        announce(f"replay {order}")
        for i in order:
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        want = [c.step() for c in sets]
        torch.cuda.synchronize()
        for i in order:
            assert same(held[i], want[i]), (order, i)


def test_two_streams():
    sets = [Calls(s) for s in (3, 4)]
    want = [c.step() for c in sets]
    torch.cuda.synchronize()
    announce("two streams at once")
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(3):
        for i, c in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.step())
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert same(g, want[i])


def test_calls_repeat():
    """No result depends on what a workspace held: large calls before small ones and back."""
    a, b = Calls(5), Calls(6)
    announce("repeated")
    first = a.step()
    b.x = {900: torch.randn(900, 2048, device=DEV) * 1e30}
    b.step()
    assert same(a.step(), first)


def test_captured_training_step():
    """A router, its loss and an MXFP4 layer's gradient in one graph, an eager graph of other
    leaves alive beside it."""
    gen = torch.Generator().manual_seed(7)
    rnd = lambda *s: torch.randn(s, generator=gen).to(DEV)                  # noqa: E731
    w = mmfp4.mxfp4_quantize(rnd(64, 256) * 0.05)
    x0 = rnd(40, 256)

    def step(x):
        y = mmfp4.mxfp4_gemm(x, *w)
        p, _ = mmfp4.moe_route(y, 4, num_groups=4, topk_groups=2)
        return torch.autograd.grad((p * p).sum() + y.square().mean(), x)[0]

    x = x0.clone().requires_grad_(True)
    alive = mmfp4.mxfp4_gemm(x0.clone().requires_grad_(True), *w)           # an eager graph
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(x)
    torch.cuda.current_stream().wait_stream(s)
    announce("capture of a training step")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(x)
    for _ in range(3):
        with torch.no_grad():
            x.copy_(rnd(40, 256))
        graph.replay()
        want = step(x.detach().clone().requires_grad_(True))
        torch.cuda.synchronize()
        assert torch.equal(held, want)
    alive.sum().backward()


@pytest.mark.parametrize("m", [0, 1, 5, 17, 33, 65, 600])
def test_sliced_operands(m):
    """Rows of a wider tensor, storage that begins off 16 bytes, and transposed layouts."""
    announce(f"sliced operands m={m}")
    gen = torch.Generator().manual_seed(8)
    rnd = lambda *s: torch.randn(s, generator=gen).to(DEV)                  # noqa: E731
    words, scales = mmfp4.mxfp4_quantize(rnd(96, 320) * 0.05)
    x = rnd(m, 320).half()
    want = mmfp4.mxfp4_gemm(x, words, scales)
    off = torch.empty(m * 320 + 1, dtype=torch.float16, device=DEV)[1:].view(m, 320).copy_(x)
    w1 = torch.empty(words.numel() + 1, dtype=torch.int32, device=DEV)[1:].view(96, 40).copy_(words)
    s1 = torch.empty(scales.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(96, 10).copy_(scales)
    assert torch.equal(mmfp4.mxfp4_gemm(off, w1, s1), want)
    assert torch.equal(mmfp4.mxfp4_gemm(x.t().contiguous().t(), words, scales), want)
    dy = rnd(m, 96).half()
    want = mmfp4.mxfp4_gemm_backward(dy, words, scales)
    assert torch.equal(mmfp4.mxfp4_gemm_backward(torch.cat([dy, dy], 1)[:, 96:], w1, s1), want)


def test_long_rows():
    """K so long that a block's scales do not fit LDS, and more values than 2^31."""
    gen = torch.Generator(DEV).manual_seed(9)
    K = 70400
    w = mmfp4.mxfp4_quantize(torch.randn(32, K, generator=gen, device=DEV) * 0.01)
    x = torch.randn(60, K, generator=gen, device=DEV)
    ref = mmfp4.mxfp4_dequantize(*mmfp4.mxfp4_quantize(x), torch.float32).double() @ \
        mmfp4.mxfp4_dequantize(*w, torch.float32).double().t()
    for m in (1, 10, 20, 60):
        announce(f"long rows m={m}")
        got = mmfp4.mxfp4_gemm(x[:m], *w).double()
        # fp32 sums of K terms of both signs, in trees of at least 64: far below 2^-16 of the norm
        assert float((got - ref[:m]).norm() / ref[:m].norm()) < 2.0 ** -16
    del x, ref
    rows, K = (1 << 31) // 512 + 3, 512
    big = torch.zeros(rows, K, dtype=torch.bfloat16, device=DEV)
    big[-3:] = torch.randn(3, K, generator=gen, device=DEV).bfloat16()
    announce("more than 2^31 values")
    words, scales = mmfp4.mxfp4_quantize(big)
    tail = mmfp4.mxfp4_quantize(big[-3:].contiguous())
    assert torch.equal(words[-3:], tail[0]) and torch.equal(scales[-3:], tail[1])
    back = mmfp4.mxfp4_dequantize(words, scales, torch.bfloat16)
    assert torch.equal(back[-3:], mmfp4.mxfp4_dequantize(*tail, torch.bfloat16))
    del back, words, scales
    w = mmfp4.mxfp4_quantize(torch.randn(40, K, generator=gen, device=DEV) * 0.05)
    y = mmfp4.mxfp4_gemm(big, *w)
    assert torch.equal(y[-3:], mmfp4.mxfp4_gemm(big[-300:], *w)[-3:])
