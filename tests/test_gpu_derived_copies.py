"""Padded and rearranged copies of weights, made at a first call: on streams that do not wait for
one another, and where that first call is captured."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from mmfp4.layers import MMFP4Linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
K, G = 1024, 64


def fresh(seed, N):
    """Weights that no call has seen, and calls that need a copy of them."""
    gen = torch.Generator().manual_seed(seed)
    w = (torch.randn((N, K), generator=gen) * 0.05).half().to(DEV)
    rnd = lambda *s: torch.randn(s, generator=gen).half().to(DEV)          # noqa: E731
    words, scales = mmfp4.quantize_fp4(w, group_size=G)
    w4, s4, z4 = mmfp4.pack_u4_weights(w, group_size=G)
    rows = MMFP4Linear(words.t().contiguous(), scales.clone(), None, G)
    rows2 = words.t().contiguous()
    ops = {"x": rnd(5, K), "dy": rnd(40, N), "gu": rnd(40, 2 * N), "words": words,
           "scales": scales, "w4": w4, "s4": s4, "z4": z4, "rows": rows2, "layer": rows}
    pair = (words, scales, words, scales)
    calls = [lambda: mmfp4.marlin_gemm_fp4_backward(ops["dy"], words, scales, G),
             lambda: mmfp4.marlin_gemm_int4_backward(ops["dy"], w4, s4, z4, G),
             lambda: mmfp4.mmfp4_gemm_rowpacked_backward(ops["dy"], rows2, scales, G),
             lambda: mmfp4.fused_gate_up_swiglu_backward(ops["dy"], ops["gu"], *pair, G),
             lambda: mmfp4.marlin_gemm_fp4(ops["x"], words, scales, G),
             lambda: mmfp4.marlin_gemm_int4(ops["x"], w4, s4, z4, G),
             lambda: rows(ops["x"])]
    return ops, calls


def expected(seed, N):
    """On weights of its own, one stream, waited for."""
    got = []
    for f in fresh(seed, N)[1]:
        got.append(f())
        torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("N", [1003, 1004])
def test_first_calls_on_two_streams(N):
    want = expected(1, N)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    busy = torch.randn((4096, 4096), device=DEV)
    ops, calls = fresh(1, N)
    torch.cuda.synchronize()
    got = []
    for i, f in enumerate(calls):
        with torch.cuda.stream(a):
            for _ in range(8):
                busy @ busy                      # the copies are made behind this
            got.append((i, f()))
        with torch.cuda.stream(b):
            got.append((i, f()))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i]), i


@pytest.mark.parametrize("N", [1003, 1004])
def test_first_call_captured(N):
    """Eager calls and a second graph come before the first graph's replay."""
    want = expected(2, N)
    ops, calls = fresh(2, N)
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append([f() for f in calls])
    for i, f in enumerate(calls):
        assert torch.equal(f(), want[i]), i
    graphs.append(torch.cuda.CUDAGraph())        # with copies that are there
    torch.cuda.synchronize()
    with torch.cuda.graph(graphs[-1]):
        held.append([f() for f in calls])
    for g in (1, 2, 0, 1, 2):
        for t in held[g]:
            t.zero_()
        graphs[g].replay()
        torch.cuda.synchronize()
        for i, y in enumerate(held[g]):
            assert torch.equal(y, want[i]), (g, i)


def test_weights_written_after_a_capture():
    """The graph's copies stay what they were; eager calls see the new weights."""
    N = 1003
    want = expected(3, N)
    ops, calls = fresh(3, N)
    for f in calls:
        f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [f() for f in calls[:2]]
    for s in (ops["scales"], ops["s4"]):
        s.mul_(2)
    for f, w in zip(calls[:2], want):
        # a power of two: the same roundings, but for halves of the smallest fp16 step
        assert ((f().double() - 2 * w.double()).abs() <= 2.0 ** -23).all()
    torch.cuda.empty_cache()
    graph.replay()
    torch.cuda.synchronize()
    for y, w in zip(held, want):
        assert torch.equal(y, w)


def test_weights_are_saved_and_copied_as_before(tmp_path):
    import copy
    ops, calls = fresh(4, 1003)
    want = [f() for f in calls]
    torch.save({k: ops[k] for k in ("words", "scales")}, tmp_path / "w.pt")
    back = torch.load(tmp_path / "w.pt", weights_only=True)
    assert torch.equal(mmfp4.marlin_gemm_fp4_backward(ops["dy"], back["words"], back["scales"], G),
                       want[0])
    layer = copy.deepcopy(ops["layer"])
    assert torch.equal(layer(ops["x"]), want[-1])
