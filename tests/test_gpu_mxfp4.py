"""MXFP4 quantization and product against their definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import DEV, announce
from mx_reference import check, half_step, quantize, rounded, sum_error, values

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed=0):
    return torch.Generator(DEV).manual_seed(seed)


def normal(*shape, dtype=torch.float32, std=1.0, seed=0):
    return (torch.randn(shape, generator=gen(seed), device=DEV) * std).to(dtype)


def spread(rows, k, dtype, seed=0):
    """Values over the type's whole range: a power of two per block, and in it ties, values at
    the ends of the codes and below the smallest."""
    g = gen(seed)
    info = torch.finfo(dtype)
    lo, hi = (-149, 127) if dtype != torch.float16 else (-24, 15)
    if dtype == torch.bfloat16:
        lo = -133
    e = torch.randint(lo, hi, (rows, k // 32, 1), generator=g, device=DEV)
    v = torch.rand((rows, k // 32, 32), generator=g, device=DEV, dtype=torch.float64) * 2 - 1
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 0.0], device=DEV,
                        dtype=torch.float64) / 8
    pick = ties[torch.randint(0, 10, v.shape, generator=g, device=DEV)]
    v = torch.where(torch.rand(v.shape, generator=g, device=DEV) < 0.3, pick * torch.sign(v), v)
    x = (v * torch.exp2(e.double() + 1)).reshape(rows, k)
    return x.clamp(-info.max, info.max).to(dtype)


def weight(n, k, seed=1):
    return quantize(normal(n, k, std=0.02, seed=seed))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (7, 1024), (65, 2048), (300, 4128)])
def test_quantize_and_back(rows, k, dtype):
    announce(f"mxfp4_quantize {rows} x {k} {dtype}")
    x = spread(rows, k, dtype, seed=rows)
    words, scales = mmfp4.mxfp4_quantize(x)
    w, s = quantize(x)
    assert words.dtype == torch.int32 and scales.dtype == torch.uint8
    assert torch.equal(scales, s)
    assert torch.equal(words, w)
    for out in TYPES:
        ref = values(w, s)
        got = mmfp4.mxfp4_dequantize(words, scales, out)
        assert got.dtype == out
        assert torch.equal(got, ref.to(out)), out       # torch rounds 64 bits to nearest, once
    assert torch.equal(mmfp4.mxfp4_dequantize(words, scales, torch.bfloat16).double(),
                       values(w, s))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_every_16_bit_pattern(dtype):
    announce(f"mxfp4_quantize patterns {dtype}")
    bits = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16)
    x = bits.view(dtype) if dtype != torch.float32 else bits.view(torch.bfloat16).float()
    x = x[torch.isfinite(x)]
    x = x[:x.numel() // 32 * 32]
    for order in (x, x[torch.randperm(x.numel(), generator=gen(3), device=DEV)]):
        rows = order.view(-1, 32)
        w, s = quantize(rows)
        words, scales = mmfp4.mxfp4_quantize(rows)
        assert torch.equal(scales, s) and torch.equal(words, w)


@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite(dtype):
    announce(f"mxfp4 not finite {dtype}")
    x = normal(4, 128, dtype=dtype)
    x[0, 5] = float("nan")
    x[1, 40] = float("inf")
    x[2, 127] = -float("inf")
    x[2, 0:32] = 0.0
    words, scales = mmfp4.mxfp4_quantize(x)
    bad = torch.zeros(4, 4, dtype=torch.bool, device=DEV)
    bad[0, 0] = bad[1, 1] = bad[2, 3] = True
    assert torch.equal(scales == 255, bad)
    assert int(scales[2, 0]) == 0
    for out in TYPES:
        v = mmfp4.mxfp4_dequantize(words, scales, out)
        assert torch.equal(torch.isnan(v), bad.repeat_interleave(32, 1))
    # a NaN row of x gives a NaN row of results, a NaN row of weights a NaN column; no others
    w, s = weight(40, 128)
    s[7, 2] = 255
    for m in (4, 36, 132):
        y = mmfp4.mxfp4_gemm(x.repeat(m // 4, 1), w, s)
        want = torch.zeros(m, 40, dtype=torch.bool, device=DEV)
        want[bad.any(1).repeat(m // 4)] = True
        want[:, 7] = True
        assert torch.equal(torch.isnan(y), want), m


def gemm_case(m, n, k, dtype, out_dtype=None, seed=0):
    x = normal(m, k, dtype=dtype, seed=seed)
    x[:, ::97] *= 10
    w, s = weight(n, k, seed=seed + 1)
    ref_x, ref_w = rounded(x), values(w, s)
    ref = ref_x @ ref_w.t()
    # products are exact; every instruction adds one rounding, and the waves' sums are added
    bound = sum_error(ref_x.abs() @ ref_w.abs().t(), k // 64 + 16) + \
        half_step(ref, out_dtype or dtype)
    y = mmfp4.mxfp4_gemm(x, w, s) if out_dtype is None else mmfp4.mxfp4_gemm(x, w, s, out_dtype)
    assert y.dtype == (out_dtype or dtype)
    check(y, ref, bound * (1 + 2.0 ** -8), f"{m} x {n} x {k}")


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 129, 257, 515])
@pytest.mark.parametrize("n,k", [(64, 256), (33, 32), (260, 992), (1, 2080), (500, 4096)])
def test_gemm(m, n, k):
    announce(f"mxfp4_gemm {m} x {n} x {k}")
    gemm_case(m, n, k, TYPES[(m + n) % 3], seed=m)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("m", [3, 24, 200])
def test_gemm_types(m, dtype, out_dtype):
    announce(f"mxfp4_gemm {m} {dtype} -> {out_dtype}")
    gemm_case(m, 132, 640, dtype, out_dtype)


@pytest.mark.parametrize("m,n,k", [(5, 14336, 4096), (48, 4096, 14336), (2048, 4096, 1024),
                                   (1000, 6144, 4096), (4100, 4099, 544)])
def test_gemm_large(m, n, k):
    announce(f"mxfp4_gemm {m} x {n} x {k}")
    gemm_case(m, n, k, torch.bfloat16)


@pytest.mark.parametrize("m", [6, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("n,k", [(8193, 5056), (8221, 736), (14336, 4096)])
def test_gemm_wide(m, n, k):
    announce(f"mxfp4_gemm {m} x {n} x {k}")
    gemm_case(m, n, k, TYPES[(m + n) % 3], seed=m)


@pytest.mark.parametrize("k", range(32, 800, 32))
def test_gemm_every_tail(k):
    announce(f"mxfp4_gemm k={k}")
    for m in (4, 20, 140):
        gemm_case(m, 72, k, torch.float16, seed=k)


def test_gemm_range():
    """Scales at both ends.  A result is finite where the sum of its terms' magnitudes, which
    bounds every partial sum, is; it is not where its value is beyond fp32; in between a partial
    sum may have left the range, whatever the order."""
    announce("mxfp4_gemm range")
    x = normal(20, 256, dtype=torch.float32)
    for row, e in enumerate(range(-120, 120, 12)):
        x[row] *= 2.0 ** e
    w, s = weight(48, 256)
    s[::2] = 1
    s[1::2] = 200
    most = torch.finfo(torch.float32).max
    for m in (16, 20):
        rx, rw = rounded(x[:m]), values(w, s)
        ref, mags = rx @ rw.t(), rx.abs() @ rw.abs().t()
        # partial sums may leave fp32's normal range at the small end: off by a subnormal step
        bound = sum_error(mags, 32) + half_step(ref, torch.float32) + 64 * 2.0 ** -149
        safe = mags * (1 + 2.0 ** -18) < most
        y = mmfp4.mxfp4_gemm(x[:m], w, s)
        assert not torch.isfinite(y[ref.abs() > most * (1 + 2.0 ** -18)]).any()
        check(torch.where(safe, y.double(), 0.0), torch.where(safe, ref, 0.0), bound)


def test_gemm_operands():
    announce("mxfp4_gemm operands")
    w, s = weight(96, 512)
    x = normal(2, 3, 5, 512, dtype=torch.bfloat16)
    y = mmfp4.mxfp4_gemm(x, w, s)
    assert y.shape == (2, 3, 5, 96)
    flat = mmfp4.mxfp4_gemm(x.view(30, 512), w, s)
    assert torch.equal(y.view(30, 96), flat)
    # columns of a wider tensor, rows in steps, a transposed one, an odd offset: same values
    wide = torch.zeros(30, 1024, dtype=torch.bfloat16, device=DEV)
    wide[:, 512:] = x.view(30, 512)
    assert torch.equal(mmfp4.mxfp4_gemm(wide[:, 512:], w, s), flat)
    turned = x.view(30, 512).t().contiguous().t()
    assert torch.equal(mmfp4.mxfp4_gemm(turned, w, s), flat)
    odd = torch.zeros(30 * 512 + 3, dtype=torch.bfloat16, device=DEV)
    odd[3:] = x.flatten()
    assert torch.equal(mmfp4.mxfp4_gemm(odd[3:].view(30, 512), w, s), flat)
    assert torch.equal(mmfp4.mxfp4_quantize(odd[3:].view(30, 512))[0],
                       mmfp4.mxfp4_quantize(x.view(30, 512))[0])
    # weights as a slice of stacked ones, unsigned words, the scale type of torch
    stacked, scales = torch.cat([w, w]), torch.cat([s, s])
    assert torch.equal(mmfp4.mxfp4_gemm(x, stacked[96:], scales[96:]), y)
    assert torch.equal(mmfp4.mxfp4_gemm(x, w.view(torch.uint32), s), y)
    if hasattr(torch, "float8_e8m0fnu"):
        assert torch.equal(mmfp4.mxfp4_gemm(x, w, s.view(torch.float8_e8m0fnu)), y)
    assert mmfp4.mxfp4_gemm(x[:0], w, s).shape == (0, 3, 5, 96)
    assert mmfp4.mxfp4_gemm(x, w[:0], s[:0]).shape == (2, 3, 5, 0)
    words, sc = mmfp4.mxfp4_quantize(x[:0])
    assert words.shape == (0, 3, 5, 64) and sc.shape == (0, 3, 5, 16)
    assert mmfp4.mxfp4_dequantize(words, sc).shape == (0, 3, 5, 512)


def test_rows_do_not_depend_on_others():
    """A row's result is that of the row alone among any rows of its kernel."""
    announce("mxfp4_gemm rows")
    w, s = weight(96, 1024)
    x = normal(300, 1024, dtype=torch.float16)
    for a, b in ((3, 16), (20, 30), (40, 64), (70, 130)):
        y = mmfp4.mxfp4_gemm(x[:b], w, s)
        other = x[:b].clone()
        other[a:] = float("inf")
        assert torch.equal(mmfp4.mxfp4_gemm(other, w, s)[:a], y[:a])
