"""Calls captured into graphs that share a capture stream (torch.cuda.graph's own): every graph
has a workspace of its own, whichever is captured or replayed first, and eager calls on that
stream are not touched by it."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16 = torch.float16


def matrix(gen, N, K, g):
    w = (torch.randn((N, K), generator=gen) * 0.05).half().to(DEV)
    return mmfp4.quantize_fp4(w, group_size=g)


class Calls:
    """Products that split their sums, forward and backward: few rows, mid-sized and prefill
    tiles, row-packed words, q/k/v, a gated block of two products (K % 64 != 0), a router, and a
    layer with adapters trained."""

    def __init__(self, seed):
        gen = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(s, generator=gen).to(DEV, F16)        # noqa: E731
        self.deep, self.g = matrix(gen, 512, 8192, 128), 128
        self.x = {m: rnd(m, 8192) for m in (1, 20, 48, 300)}
        self.rows = self.deep[0].t().contiguous()
        self.pair = matrix(gen, 256, 96, 32)
        self.a, self.dh = rnd(50, 96), rnd(50, 256)
        self.h, self.gate = rnd(4, 2048), rnd(2048, 64)
        self.layer = mmfp4.LoRALinear(mmfp4.MarlinLinear(*self.deep, None, self.g), 8, 3, 0.5)
        with torch.no_grad():
            self.layer.lora_b.copy_(rnd(*self.layer.lora_b.shape))
        self.ids = torch.randint(-1, 3, (300,), generator=gen).to(DEV)

    def step(self):
        out = [mmfp4.marlin_gemm_fp4(x, *self.deep, self.g) for x in self.x.values()]
        out += [mmfp4.mmfp4_gemm_rowpacked(x, self.rows, self.deep[1], self.g)
                for x in self.x.values()]
        out += mmfp4.mmfp4_fused_qkv(self.x[20], *self.deep * 3, self.g)
        h, kept = mmfp4.fused_gate_up_swiglu(self.a, *self.pair * 2, 32)
        out += [h, kept, mmfp4.fused_gate_up_swiglu_backward(self.dh, kept, *self.pair * 2, 32)]
        out += mmfp4.moe_router_topk(self.h, self.gate, 4)
        x = self.x[300].requires_grad_(True)
        y = self.layer(x, self.ids)
        out += torch.autograd.grad(y, (x, *self.layer.parameters()), y.detach() * 1e-2)
        x.requires_grad_(False)
        return [y.detach(), *out]

    def renew(self, gen):
        for x in (*self.x.values(), self.a, self.dh, self.h):
            x.copy_(torch.randn(x.shape, generator=gen))


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("binding", [True, False])
def test_graphs_of_one_stream(binding, monkeypatch):
    """Captured cold on one stream, the second replayed first, then both at once; through the
    per-call binding and through ctypes."""
    if not binding:
        monkeypatch.setattr("mmfp4._lib._binding", False)
        monkeypatch.setattr("mmfp4.kernels._BINDING", False)
    sets = [Calls(s) for s in (1, 2)]
    for c in sets:
        c.step()                                    # on the current stream, not the capture's
    torch.cuda.synchronize()
    mmfp4.release_workspaces()
    graphs, held = [], []
    for c in sets:
        announce("capture")
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(c.step())
    gen = torch.Generator().manual_seed(3)
    streams = [torch.cuda.Stream() for _ in sets]
    for order in ([1], [0], [0, 1], [1, 0], [0, 1]):
        for c in sets:
            c.renew(gen)
        torch.cuda.synchronize()
        announce(f"replay {order}")
        for i in order:
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        want = [c.step() for c in sets]             # eager calls beside them
        torch.cuda.synchronize()
        for i in order:
            assert same(held[i], want[i]), (order, i)


def test_eager_calls_on_the_capture_stream():
    """A workspace first needed under capture is not the stream's own afterwards."""
    c = Calls(4)
    want = c.step()
    torch.cuda.synchronize()
    mmfp4.release_workspaces()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        held = c.step()
    with torch.cuda.stream(s):
        got = c.step()                              # the graph has not been replayed yet
    torch.cuda.synchronize()
    assert same(got, want)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert same(held, want)
    del graph, held
    with torch.cuda.stream(s):
        assert same(c.step(), want)


def test_capture_ids():
    from mmfp4 import _lib
    s, seen = torch.cuda.Stream(), set()
    x = torch.zeros(8, device=DEV)
    assert _lib.load().mm_capture_id(s.cuda_stream) == 0
    for _ in range(3):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            x.add_(1)
            here = _lib.load().mm_capture_id(s.cuda_stream)
            assert here == _lib.load().mm_capture_id(s.cuda_stream)
            seen.add(here)
    assert len(seen) == 3 and 0 not in seen
