"""Input gradients, the gated block and adapters as a program may call them: on several streams
at once, in graphs that replay at once, and on tensors of more than 2^31 elements."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


class Operands:
    """Sizes at which every call splits its sums (workspaces with counters)."""

    def __init__(self, seed, dtype=BF16, T=260, K=512, N=2048, g=64, r=16, L=3):
        gen = torch.Generator().manual_seed(seed)
        rnd = lambda *s, std=1.0: (torch.randn(s, generator=gen) * std).to(DEV, dtype)  # noqa
        mats = [mmfp4.quantize_fp4(rnd(N, K, std=0.05).half(), group_size=g) for _ in range(2)]
        self.mats, self.g = [t for m in mats for t in m], g
        self.x, self.dy, self.one = rnd(T, K), rnd(T, N, std=1e-2), rnd(1, N, std=1e-2)
        self.a, self.b = rnd(L, r, K, std=0.05), rnd(L, N, r, std=0.05)
        self.ids = torch.randint(-1, L, (T,), generator=gen).to(DEV)

    def step(self):
        m = self.mats
        h, pair = mmfp4.fused_gate_up_swiglu(self.x, *m, self.g)
        dx = mmfp4.fused_gate_up_swiglu_backward(self.dy, pair, *m, self.g)
        one = mmfp4.marlin_gemm_fp4_backward(self.one, *m[:2], self.g)
        y = mmfp4.lora_add(h, self.x, self.a, self.b, self.ids, 0.5)
        few = mmfp4.lora_add(h[:3], self.x[:3], self.a, self.b, self.ids[:3], 0.5)
        return (h, pair, one, y, few, *mmfp4.lora_backward(self.dy, self.x, self.a, self.b,
                                                           self.ids, 0.5, dx_base=dx))


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    ops = [Operands(s) for s in (1, 2)]
    want = [o.step() for o in ops]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ops]
    got = [[], []]
    for _ in range(6):
        for o, s, out in zip(ops, streams, got):
            with torch.cuda.stream(s):
                out.append(o.step())
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(same(o, w) for o in outs)


def test_two_graphs_at_once():
    """Of the same call on the same operands, replayed on two streams without a wait between."""
    o = Operands(3)
    streams, graphs, held = [torch.cuda.Stream() for _ in range(2)], [], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.stream(s):
            o.step()
            with torch.cuda.graph(graphs[-1], stream=s):
                held.append(o.step())
    torch.cuda.synchronize()
    gen = torch.Generator().manual_seed(4)
    for i in range(4):
        o.x.copy_(torch.randn(o.x.shape, generator=gen))
        o.dy.copy_(torch.randn(o.dy.shape, generator=gen) * 1e-2)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        want = o.step()
        torch.cuda.synchronize()
        assert same(held[0], want) and same(held[1], want), i


def test_operands_of_another_stream():
    """Made on one stream, used on another that waits for it, freed at once."""
    o = Operands(5)
    want = o.step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    x = o.x
    for _ in range(4):
        o.x = (x * 2) / 2                  # on the current stream
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = o.step()
        o.x.record_stream(s)
        o.x = x
        torch.cuda.current_stream().wait_stream(s)
        assert same(got, want)


def test_adapters_past_2_31_elements():
    """The last 70 of 140000 tokens have values; the same 70 by themselves are the reference. Each
    of the two is off by half a step of the result, by 2^-16 of H (hi + lo in bf16) and by the
    order of its fp32 sums."""
    T, n, K, N, r = 140_000, 70, 64, 16384, 8
    announce(f"adapters {T} {K} {N}")
    gen = torch.Generator().manual_seed(6)
    rnd = lambda *s: torch.randn(s, generator=gen).to(DEV, BF16)          # noqa: E731
    x, base, dy = (torch.zeros((T, c), device=DEV, dtype=BF16) for c in (K, N, N))
    assert base.numel() > 2 ** 31
    for t in (x, base, dy):
        t[-n:] = rnd(n, t.shape[1])
    a, b = rnd(2, r, K), rnd(2, N, r)
    ids = torch.full((T,), -1, dtype=torch.int32, device=DEV)
    ids[-n:] = torch.arange(n, device=DEV) % 2
    tail = [t[-n:].clone() for t in (base, x, ids, dy)]

    def close(got, ref, mags, terms):
        tol = 2 * torch.finfo(BF16).eps / 2 * ref.abs() + \
            (2.0 ** -15 + 2 * terms * 2.0 ** -23) * mags
        return ((got.double() - ref).abs() <= tol + 1e-30).all()

    out = mmfp4.lora_add(base, x, a, b, ids)
    small = mmfp4.lora_add(tail[0], tail[1], a, b, tail[2])
    pick = lambda w: w.double().abs()[tail[2].long()]                      # noqa: E731
    h = torch.bmm(pick(a), tail[1].double().abs().unsqueeze(2))            # magnitudes [n, r, 1]
    mags = torch.bmm(pick(b), h).squeeze(2) + tail[0].double().abs()
    assert not out[:-n].any() and close(out[-n:], small.double(), mags, K + r)
    del out
    dx, da, db = mmfp4.lora_backward(dy, x, a, b, ids)
    sx, sa, sb = mmfp4.lora_backward(tail[3], tail[1], a, b, tail[2])
    dh = torch.bmm(tail[3].double().abs().unsqueeze(1), pick(b))           # [n, 1, r]
    assert not dx[:-n].any()
    assert close(dx[-n:], sx.double(), torch.bmm(dh, pick(a)).squeeze(1), N + r)
    for e in range(2):
        k = tail[2] == e
        ma = dh[k].squeeze(1).t() @ tail[1][k].double().abs()
        mb = tail[3][k].double().abs().t() @ h[k].squeeze(2)
        assert close(da[e], sa[e].double(), ma, N + n)
        assert close(db[e], sb[e].double(), mb, K + n)


def test_input_gradients_past_2_31_elements():
    """Rows do not depend on one another: the last ones by themselves are the reference, up to
    the order of fp32 sums (256 terms) and half a step of the result each."""
    M, n, K, N, g = 140_000, 64, 16384, 128, 128
    announce(f"input gradients {M} {N} {K}")
    gen = torch.Generator().manual_seed(7)
    m = [t for _ in range(2) for t in
         mmfp4.quantize_fp4((torch.randn((N, K), generator=gen) * 0.05).half().to(DEV),
                            group_size=g)]
    dy = torch.zeros((M, N), device=DEV, dtype=BF16)
    dy[-n:] = torch.randn((n, N), generator=gen).to(DEV, BF16)
    W = [mmfp4.dequant_fp4(m[i], m[i + 1], K, N, g).double() for i in (0, 2)]

    def close(got, ref, mags):
        tol = 2 * torch.finfo(BF16).eps / 2 * ref.abs() + 512 * 2.0 ** -23 * mags
        return ((got.double() - ref).abs() <= tol + 1e-30).all()

    out = mmfp4.marlin_gemm_fp4_backward(dy, *m[:2], g)
    assert out.numel() > 2 ** 31 and not out[:-n].any()
    ref = mmfp4.marlin_gemm_fp4_backward(dy[-n:].clone(), *m[:2], g)
    assert close(out[-n:], ref.double(), dy[-n:].double().abs() @ W[0].abs().t())
    del out
    pair = torch.zeros((M, 2 * N), device=DEV, dtype=F16)
    pair[-n:] = torch.randn((n, 2 * N), generator=gen).to(DEV, F16)
    out = mmfp4.fused_gate_up_swiglu_backward(dy, pair, *m, g)
    ref = mmfp4.fused_gate_up_swiglu_backward(dy[-n:].clone(), pair[-n:].clone(), *m, g)
    # |dg| <= 1.1 |dh u|, |du| <= |dh g|
    G, U = pair[-n:].double().abs().split(N, 1)
    D = dy[-n:].double().abs()
    mags = (1.1 * D * U) @ W[0].abs().t() + (D * G) @ W[1].abs().t()
    assert not out[:-n].any() and close(out[-n:], ref.double(), mags)
