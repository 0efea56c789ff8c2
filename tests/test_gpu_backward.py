"""Input gradients of the quantized products and the gate/up block with its backward pass,
against the formulas in 64 bits.

Tolerances are error bounds, element by element.  A product over n terms in fp32 is off by at
most n * 2^-23 of the sum of its terms' magnitudes, and its result by half a step of its type.
bf16 and fp32 gradients and those inside the block are carried in fp16 under one power of two
per row: a value v of a row with maximum m is off by at most 2^-12 |v| rounded up to half a
step, 2^-11 |v| (nothing for bf16, whose 8 bits fit), or by 2^-40 m where it is subnormal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mmfp4
from gpu_helpers import announce
from oracle import fp4 as ofp4

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def half_step(t):
    return torch.finfo(t).eps / 2


def make_fp4(gen, K, N, g, rows=False):
    """(words, scales, W [K, N] in 64 bits)."""
    w = (torch.randn((N, K), generator=gen) * 0.05).half().numpy()
    packed, scales = ofp4.quantize_fp4(w, g)
    W = torch.from_numpy(ofp4.dequant_fp4(packed, scales, g).astype(np.float64)).to(DEV)
    words = torch.from_numpy(packed.view(np.int32)).to(DEV)
    return (words.t().contiguous() if rows else words), torch.from_numpy(scales).to(DEV), W


def make_int4(gen, K, N, g):
    w = (torch.randn((N, K), generator=gen) * 0.05).half()
    words, scales, zeros = mmfp4.pack_u4_weights(w.to(DEV), group_size=g)
    W = mmfp4.dequant_int4(words, scales, zeros, K, N, g).double()
    return words, scales, zeros, W


def check(out, ref, terms, n, dtype, carried=0.0, what=""):
    """terms: the sum of the terms' magnitudes; carried: error of the operands, summed."""
    assert out.dtype == dtype and out.shape == ref.shape, (what, out.dtype, out.shape)
    tiny = torch.finfo(dtype).smallest_normal * half_step(dtype)
    tol = (half_step(dtype) * (1 + 1e-3)) * ref.abs() + tiny + n * 2.0 ** -23 * terms + carried
    off = (out.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst " \
        f"{float((off / tol).max())} of the bound"


def check_linear(out, dC, W, dtype, what):
    d = dC.double()
    carried = 0.0
    if dC.dtype != F16:
        m = d.abs().amax(1, keepdim=True)
        step = 2.0 ** -11 * d.abs() if dC.dtype == F32 else 0.0
        carried = (step + 2.0 ** -40 * m + 0 * d) @ W.abs().t()
    check(out, d @ W.t(), d.abs() @ W.abs().t(), W.shape[1] + 8, dtype, carried, what)


SHAPES = [  # M, N, K, g
    (1, 64, 64, 32), (1, 4096, 1024, 128), (2, 8, 8, 8), (3, 72, 264, 8), (17, 136, 1032, 24),
    (31, 1000, 256, 16), (33, 520, 512, 64), (64, 6, 768, 128), (65, 200, 520, 40),
    (100, 1024, 2048, 256), (129, 328, 1280, 128), (200, 35, 288, 32), (300, 2048, 544, 32),
    (513, 648, 320, 64),
]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K,g", SHAPES)
def test_fp4(M, N, K, g, dtype):
    announce(f"fp4 backward {M} {N} {K} {g} {dtype}")
    gen = torch.Generator().manual_seed(M + N + K)
    words, scales, W = make_fp4(gen, K, N, g)
    dC = torch.randn((M, N), generator=gen).to(DEV, dtype)
    check_linear(mmfp4.marlin_gemm_fp4_backward(dC, words, scales, g), dC, W, dtype, "fp4")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K,g", SHAPES)
def test_int4(M, N, K, g, dtype):
    announce(f"int4 backward {M} {N} {K} {g} {dtype}")
    gen = torch.Generator().manual_seed(M + N + K)
    words, scales, zeros, W = make_int4(gen, K, N, g)
    dC = torch.randn((M, N), generator=gen).to(DEV, dtype)
    check_linear(mmfp4.marlin_gemm_int4_backward(dC, words, scales, zeros, g), dC, W, dtype,
                 "int4")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K,g", SHAPES)
def test_rowpacked(M, N, K, g, dtype):
    announce(f"rowpacked backward {M} {N} {K} {g} {dtype}")
    gen = torch.Generator().manual_seed(M + N + K)
    words, scales, W = make_fp4(gen, K, N, g, rows=True)
    dC = torch.randn((M, N), generator=gen).to(DEV, dtype)
    out = mmfp4.mmfp4_gemm_rowpacked_backward(dC, words, scales, g)
    check_linear(out, dC, W, dtype, "rows")
    if N != K // g:
        again = mmfp4.mmfp4_gemm_rowpacked_backward(dC, words, scales.t().contiguous(), g)
        assert torch.equal(out, again)
    marlin = mmfp4.marlin_gemm_fp4_backward(dC, words.t().contiguous(), scales, g)
    assert torch.equal(out, marlin)


# Sizes at which the time model takes each tile (64 x 128, 64 x 256, 256 x 256), whole and split,
# with chunks that end inside a tile, small groups and large.
TILES = [(64, 2056, 480, 8), (256, 2056, 480, 48), (70, 4104, 96, 96), (64, 8200, 480, 24),
         (256, 8200, 480, 32), (1000, 264, 2080, 8), (1030, 520, 2080, 104), (2050, 200, 4096, 16),
         (2050, 520, 4096, 64), (1000, 8200, 2080, 32)]


@pytest.mark.parametrize("fmt", ["fp4", "int4", "rows"])
@pytest.mark.parametrize("M,N,K,g", TILES)
def test_tiles(M, N, K, g, fmt):
    announce(f"tiles {M} {N} {K} {g} {fmt}")
    gen = torch.Generator().manual_seed(M + N + K)
    dC = torch.randn((M, N), generator=gen).to(DEV, F16)
    if fmt == "int4":
        words, scales, zeros, W = make_int4(gen, K, N, g)
        out = mmfp4.marlin_gemm_int4_backward(dC, words, scales, zeros, g)
    else:
        words, scales, W = make_fp4(gen, K, N, g, rows=fmt == "rows")
        call = mmfp4.mmfp4_gemm_rowpacked_backward if fmt == "rows" else \
            mmfp4.marlin_gemm_fp4_backward
        out = call(dC, words, scales, g)
    check_linear(out, dC, W, F16, fmt)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,Ns", [(1, (512, 128, 128)), (50, (72, 8, 40)), (260, (256, 65, 64))])
def test_qkv(M, Ns, dtype):
    announce(f"qkv backward {M} {Ns} {dtype}")
    K, g = 256, 64
    gen = torch.Generator().manual_seed(M)
    mats = [make_fp4(gen, K, n, g) for n in Ns]
    d = [torch.randn((M, n), generator=gen).to(DEV, dtype) * 10.0 ** i for i, n in enumerate(Ns)]
    args = [t for w, s, _ in mats for t in (w, s)]
    out = mmfp4.mmfp4_fused_qkv_backward(*d, *args, g)
    check_linear(out, torch.cat(d, 1), torch.cat([W for _, _, W in mats], 1), dtype, "qkv")


def test_range_of_bf16_gradients():
    """Rows of gradients far below what fp16 holds, or above it, in one batch; a zero row."""
    gen = torch.Generator().manual_seed(5)
    words, scales, W = make_fp4(gen, 256, 320, 64)
    mag = torch.tensor([1e-30, 1e-12, 1.0, 1e6, 1e30, 0.0]).view(-1, 1)
    dC = (torch.randn((6, 320), generator=gen) * mag).to(DEV, BF16)
    out = mmfp4.marlin_gemm_fp4_backward(dC, words, scales, 64)
    check_linear(out, dC, W, BF16, "range")
    assert not out[5].any()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_qkv_of_one_tensor(dtype):
    """The three gradients as columns of one tensor (strided views), and no rows at all: the
    per-call binding and the checked path give the same bits."""
    K, g, Ns = 256, 64, (256, 72, 64)
    gen = torch.Generator().manual_seed(9)
    mats = [make_fp4(gen, K, n, g) for n in Ns]
    args = [t for w, s, _ in mats for t in (w, s)]
    whole = torch.randn((77, sum(Ns)), generator=gen).to(DEV, dtype) * 1e-3
    views = whole.split(Ns, 1)
    out = mmfp4.mmfp4_fused_qkv_backward(*[v.contiguous() for v in views], *args, g)
    check_linear(out, whole, torch.cat([W for _, _, W in mats], 1), dtype, "qkv")
    assert torch.equal(out, mmfp4.mmfp4_fused_qkv_backward(*views, *args, g))
    none = mmfp4.mmfp4_fused_qkv_backward(*[v[:0] for v in views], *args, g)
    assert none.shape == (0, K) and none.dtype == dtype
    assert mmfp4.marlin_gemm_fp4_backward(views[0][:0], *args[:2], g).shape == (0, K)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_non_finite_rows_stay_by_themselves(dtype):
    gen = torch.Generator().manual_seed(6)
    words, scales, W = make_fp4(gen, 512, 320, 128)
    dC = torch.randn((70, 320), generator=gen).to(DEV, dtype)
    dirty = dC.clone()
    dirty[3, 5], dirty[69, 319] = float("nan"), float("inf")
    ref = mmfp4.marlin_gemm_fp4_backward(dC, words, scales, 128)
    out = mmfp4.marlin_gemm_fp4_backward(dirty, words, scales, 128)
    keep = [i for i in range(70) if i not in (3, 69)]
    assert torch.equal(out[keep], ref[keep])
    assert out[3].isnan().all() and not out[69].isfinite().any()


def test_non_finite_scales_count_as_zero():
    gen = torch.Generator().manual_seed(7)
    words, scales, W = make_fp4(gen, 256, 96, 32)
    scales[2, 10], scales[5, 95], scales[0, 0] = float("inf"), float("nan"), -float("inf")
    for grp, n in ((2, 10), (5, 95), (0, 0)):
        W[32 * grp:32 * (grp + 1), n] = 0
    dC = torch.randn((40, 96), generator=gen).to(DEV, F16)
    check_linear(mmfp4.marlin_gemm_fp4_backward(dC, words, scales, 32), dC, W, F16, "scales")


def test_forms_of_the_gradient():
    """Leading axes, strides, offsets, no rows, another output type."""
    gen = torch.Generator().manual_seed(8)
    words, scales, W = make_fp4(gen, 256, 96, 32)
    base = torch.randn((2, 5, 100), generator=gen).to(DEV, F16)
    view = base[:, :, 1:97]                                   # rows 200 bytes apart, odd start
    out = mmfp4.marlin_gemm_fp4_backward(view, words, scales, 32)
    assert out.shape == (2, 5, 256)
    flat = view.reshape(10, 96).contiguous()
    assert torch.equal(out.view(10, 256), mmfp4.marlin_gemm_fp4_backward(flat, words, scales, 32))
    off = torch.empty(961, dtype=F16, device=DEV)[1:]         # 2 bytes past a boundary
    off.copy_(flat.view(-1))
    assert torch.equal(out.view(10, 256),
                       mmfp4.marlin_gemm_fp4_backward(off.view(10, 96), words, scales, 32))
    assert mmfp4.marlin_gemm_fp4_backward(flat[:0], words, scales, 32).shape == (0, 256)
    one = mmfp4.marlin_gemm_fp4_backward(flat[0], words, scales, 32)
    assert one.shape == (256,)
    check_linear(mmfp4.marlin_gemm_fp4_backward(flat, words, scales, 32, out_dtype=F32), flat, W,
                 F32, "fp32 out")


# ------------------------------------------------------------------ the gate/up block
def silu_parts(gu):
    g, u = gu.double().chunk(2, 1)
    s = torch.sigmoid(g)
    return g, u, s


BLOCK = [(1, 64, 64, 32, F16), (1, 1408, 2048, 128, F16), (8, 40, 128, 64, BF16),
         (20, 512, 1024, 128, F16), (33, 264, 512, 64, F16), (100, 1000, 512, 128, BF16),
         (200, 72, 320, 32, F16), (300, 512, 512, 128, F32), (1100, 2048, 256, 64, F16),
         (5, 30, 64, 32, F16), (40, 36, 72, 8, F16)]


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("M,N,K,g,dtype", BLOCK)
def test_block(M, N, K, g, dtype, rows):
    announce(f"block {M} {N} {K} {g} {dtype} rows={rows}")
    gen = torch.Generator().manual_seed(M + N)
    gw, gs, Wg = make_fp4(gen, K, N, g, rows)
    uw, us, Wu = make_fp4(gen, K, N, g, rows)
    x = torch.randn((M, K), generator=gen).to(DEV, dtype)
    h, gu = mmfp4.fused_gate_up_swiglu(x, gw, gs, uw, us, g, row_packed=rows)
    # the mid-sized kernel may apply a group's scale to its sum, where the weights have not been
    # rounded to fp16: 2^-11
    xd = x.half().double()
    W = torch.cat([Wg, Wu], 1)
    terms = xd.abs() @ W.abs()
    check(gu, xd @ W, terms, K + 8, F16, 2.0 ** -11 * terms, "gate_up")
    err = (2.0 ** -11 + (K + 8) * 2.0 ** -23) * terms + 2.0 ** -11 * (xd @ W).abs() + 2.0 ** -24
    gr, ur, sr = silu_parts(xd @ W)
    eg, eu = err.chunk(2, 1)
    href = gr * sr * ur
    check(h, href, href.abs(), 16, F16,
          1.1 * eg * ur.abs() + (gr * sr).abs() * eu + 1.1 * eg * eu, "h")
    if not rows and M > 32 and N % 8 == 0 and K % 64 == 0:
        assert torch.equal(gu, mmfp4.fused_gate_up_gemm(x, gw, gs, uw, us, g))
        assert torch.equal(h, mmfp4.mmfp4_fused_gate_up_marlin(x, gw, gs, uw, us, g))
    dh = torch.randn((M, N), generator=gen).to(DEV, dtype) * 1e-3
    dx = mmfp4.fused_gate_up_swiglu_backward(dh, gu, gw, gs, uw, us, g, row_packed=rows)
    check_block_gradient(dx, dh, gu, W, dtype)


def check_block_gradient(dx, dh, gu, W, dtype):
    gr, ur, sr = silu_parts(gu)
    d = dh.double()
    dgu = torch.cat([d * ur * (sr + gr * sr * (1 - sr)), d * gr * sr], 1)
    # exp and the division in fp32: a few steps of the factors, which cancel near g = -1.28
    soft = torch.cat([d.abs() * ur.abs() * (1 + gr.abs()) * sr, d.abs() * gr.abs() * sr], 1)
    # sig is an fp32 number: below 2^-126, its smallest normal value, it counts as 0 (sig(-100) =
    # 2^-144.3 does), and dg = dh u sig (1 + g (1 - sig)), du = dh g sig are then off by less than
    # 2^-126 |dh| |u| (1 + |g|) and 2^-126 |dh| |g|
    soft = soft + 2.0 ** -106 * torch.cat([d.abs() * ur.abs(), d.abs()], 1)
    m = dgu.abs().amax(1, keepdim=True)
    e = 2.0 ** -11 * dgu.abs() + 2.0 ** -20 * (1 + gr.abs().repeat(1, 2)) * soft + 2.0 ** -40 * m
    check(dx, dgu @ W.t(), dgu.abs() @ W.abs().t(), 2 * W.shape[1], dtype, e @ W.abs().t(), "dx")


def test_block_gradient_at_extreme_gates():
    """Gates where exp overflows or underflows; rows of zeros; gradients near fp16's ends."""
    gen = torch.Generator().manual_seed(9)
    K, N, g = 256, 64, 64
    gw, gs, Wg = make_fp4(gen, K, N, g)
    uw, us, Wu = make_fp4(gen, K, N, g)
    gu = torch.randn((40, 2 * N), generator=gen)
    gu[0, :N], gu[1, :N], gu[2, :N], gu[3, :N] = 60000.0, -60000.0, -100.0, 88.0
    gu[4] = 0.0
    gu[5, N:] = 60000.0
    dh = torch.randn((40, N), generator=gen)
    dh[6] = 0.0
    dh[7] *= 1e-7
    dh[8] = 60000.0
    gu, dh = gu.to(DEV, F16), dh.to(DEV, F16)
    dx = mmfp4.fused_gate_up_swiglu_backward(dh, gu, gw, gs, uw, us, g, out_dtype=F32)
    assert dx.isfinite().all() and not dx[6].any() and not dx[1].any()
    check_block_gradient(dx, dh, gu, torch.cat([Wg, Wu], 1), F32)
    gu[9, :N] = -float("inf")                       # a masked gate: silu and its slope are 0
    dx = mmfp4.fused_gate_up_swiglu_backward(dh, gu, gw, gs, uw, us, g)
    assert not dx[9].any()


def test_block_gradient_by_differences():
    """dx against central differences of the block in 64 bits."""
    gen = torch.Generator().manual_seed(10)
    K, N, g = 64, 48, 32
    gw, gs, Wg = make_fp4(gen, K, N, g)
    uw, us, Wu = make_fp4(gen, K, N, g)
    x = torch.randn((3, K), generator=gen).to(DEV, F16)
    dh = torch.randn((3, N), generator=gen).to(DEV, F16)
    _, gu = mmfp4.fused_gate_up_swiglu(x, gw, gs, uw, us, g)
    dx = mmfp4.fused_gate_up_swiglu_backward(dh, gu, gw, gs, uw, us, g, out_dtype=F32)

    def loss(v):
        gate, up = v @ Wg, v @ Wu
        return (gate * torch.sigmoid(gate) * up * dh.double()).sum(1)
    e, xd = 1e-5, x.double()
    num = torch.stack([(loss(xd + e * torch.eye(K, device=DEV, dtype=xd.dtype)[i]) -
                        loss(xd - e * torch.eye(K, device=DEV, dtype=xd.dtype)[i])) / (2 * e)
                       for i in range(K)], 1)
    # the kept products are rounded to fp16 (2^-11) and so are their gradients
    assert float((dx.double() - num).abs().max()) <= 2.0 ** -7 * float(num.abs().max())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_capture(dtype):
    """A training step's calls captured once, replayed on new contents, eager work between."""
    gen = torch.Generator().manual_seed(11)
    K, N, g, M = 512, 256, 64, 40
    gw, gs, _ = make_fp4(gen, K, N, g)
    uw, us, _ = make_fp4(gen, K, N, g)
    x = torch.randn((M, K), generator=gen).to(DEV, dtype)
    dh = torch.randn((M, N), generator=gen).to(DEV, dtype)

    def step():
        h, gu = mmfp4.fused_gate_up_swiglu(x, gw, gs, uw, us, g)
        return h, gu, mmfp4.fused_gate_up_swiglu_backward(dh, gu, gw, gs, uw, us, g), \
            mmfp4.marlin_gemm_fp4_backward(dh, gw, gs, g)
    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        x.copy_(torch.randn((M, K), generator=gen))
        dh.copy_(torch.randn((M, N), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b), i


def test_streams_of_their_own():
    gen = torch.Generator().manual_seed(12)
    words, scales, _ = make_fp4(gen, 4096, 1024, 128)
    dCs = [torch.randn((4, 1024), generator=gen).to(DEV, F16) for _ in range(4)]
    refs = [mmfp4.marlin_gemm_fp4_backward(d, words, scales, 128) for d in dCs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dCs]
    outs = []
    for s, d in zip(streams, dCs):
        with torch.cuda.stream(s):
            outs.append([mmfp4.marlin_gemm_fp4_backward(d, words, scales, 128)
                         for _ in range(8)])
    torch.cuda.synchronize()
    for o, r in zip(outs, refs):
        assert all(torch.equal(v, r) for v in o)
