"""MXFP4 weights at the ends of their scales' range: codes 253 and 254 hold values beyond fp32 and
bf16 (4 * 2^126, 2 * 2^127), whose products with small numbers are ordinary ones all the same."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import DEV, announce
from mx_reference import check, half_step, quantize, rounded, sum_error, values

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(*shape, dtype=torch.float32, std=1.0, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def weight(n, k, code):
    """Codes of ordinary values, scale code[n] in every second block of row n, 1 in the others."""
    w, s = quantize(normal(n, k))
    s[:, 0::2] = code.to(torch.uint8).unsqueeze(1)
    s[:, 1::2] = 127
    return w, s


@pytest.mark.parametrize("dtype", TYPES)
def test_every_value(dtype):
    """All 16 codes under all 256 scales, back to values: one rounding of a type that ends where
    infinity begins."""
    announce(f"mxfp4_dequantize every value {dtype}")
    w = torch.tensor([0x76543210, -0x01234568], dtype=torch.int32, device=DEV).repeat(256, 2)
    s = torch.arange(256, device=DEV).to(torch.uint8).unsqueeze(1)
    got, want = mmfp4.mxfp4_dequantize(w, s, dtype), values(w, s).to(dtype)
    assert torch.isnan(got[255]).all() and torch.equal(got[:255], want[:255])
    assert torch.equal(torch.signbit(got[:255]), torch.signbit(want[:255]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(3, 255, 96), (40, 255, 64), (255, 255, 320), (500, 2000, 256),
                                   (33, 2041, 64)])
def test_gradient_of_every_scale(m, n, k, dtype):
    """One product per result, and zeros of dY that meet weights of every scale: exact."""
    announce(f"mxfp4_gemm_backward every scale {m} x {n} x {k} {dtype}")
    code = 254 - torch.arange(n, device=DEV) % 255
    w, s = weight(n, k, code)
    at = torch.arange(m, device=DEV) * 7 % n
    # as far from 1 as the scale is on the other side, within the type's normal range
    far = 14 if dtype == torch.float16 else 100
    e = (127 - code[at]).clamp(-far, far).double()
    # 8, 11 and 16 bits: one, two and two terms, whose products with 2 bits fp32 holds
    bits = {torch.bfloat16: 7, torch.float16: 10, torch.float32: 15}[dtype]
    one = 1 + torch.randint(0, 1 << bits, (m,), device=DEV,
                            generator=torch.Generator(DEV).manual_seed(m)) / (1 << bits)
    dy = torch.zeros(m, n, dtype=torch.float64, device=DEV)
    dy[torch.arange(m), at] = one.double() * torch.exp2(e)
    assert torch.equal(dy, dy.to(dtype).double())
    dx = mmfp4.mxfp4_gemm_backward(dy.to(dtype), w, s, torch.float32)
    ref = dy @ values(w, s)
    assert torch.isfinite(ref.float()).all()
    assert torch.equal(dx.double(), ref)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [2, 150])
def test_gradient_beyond_fp32(m, dtype):
    """What is beyond fp32 is infinite, what no such weight reaches is not."""
    announce(f"mxfp4_gemm_backward beyond fp32 {m} {dtype}")
    code = torch.full((70,), 120, device=DEV)
    code[[3, 69]] = torch.tensor([254, 253], device=DEV)
    w, s = weight(70, 64, code)
    w[3], w[69] = 0x22222222, 0x70707070                  # ones; 6 and 0 in turn
    dy = normal(m, 70, dtype=dtype)
    dy[:, 3] = dy[:, 69] = 0
    dy[0, 3], dy[1, 69] = 2, -4
    ref = dy.double() @ values(w, s)
    dx = mmfp4.mxfp4_gemm_backward(dy, w, s, torch.float32)
    big = ref.abs() > torch.finfo(torch.float32).max
    assert big[0, :32].all() and big[1, 1:32:2].all() and int(big.sum()) == 48
    assert torch.equal(dx[big].double(), torch.sign(ref[big]) * torch.inf)
    bound = sum_error(dy.double().abs() @ values(w, s).abs(), 3 * 70) + half_step(ref, torch.float32)
    check(torch.where(big, 0.0, dx.double()), torch.where(big, 0.0, ref), bound * (1 + 2.0 ** -8))


@pytest.mark.parametrize("m", [5, 150])
def test_gradient_of_small_fp32(m):
    """fp32 gradients below 2^-109, whose 24 bits reach below bf16's smallest step: less than that
    step of each is cut off, and nothing of those whose bits end above it."""
    announce(f"mxfp4_gemm_backward small fp32 {m}")
    w, s = weight(136, 96, torch.full((136,), 200, device=DEV))
    rw = values(w, s)
    dy = normal(m, 136) * torch.exp2(-100.0 - torch.arange(136, device=DEV) % 49)
    whole = (torch.trunc(dy.double() * 2.0 ** 133) * 2.0 ** -133).float()
    for dy, cut in ((dy, 2.0 ** -133 * rw.abs().sum(0)), (whole, 0.0)):
        ref = dy.double() @ rw
        bound = sum_error(dy.double().abs() @ rw.abs(), 3 * 136 // 4 + 40) + half_step(ref, torch.float32)
        check(mmfp4.mxfp4_gemm_backward(dy, w, s), ref, bound * (1 + 2.0 ** -8) + cut)


@pytest.mark.parametrize("m", [1, 20, 60, 140])
def test_product_of_the_largest_scales(m):
    announce(f"mxfp4_gemm largest scales {m}")
    w, s = weight(72, 288, 250 + torch.arange(72, device=DEV) % 5)
    for dtype in (torch.float32, torch.bfloat16):
        x = normal(m, 288, dtype=dtype, seed=m) * 2.0 ** -100
        x[:, 40:80] = 0
        rx, rw = rounded(x), values(w, s)
        ref = rx @ rw.t()
        bound = sum_error(rx.abs() @ rw.abs().t(), 288 // 64 + 16) + half_step(ref, dtype)
        check(mmfp4.mxfp4_gemm(x, w, s), ref, bound * (1 + 2.0 ** -8))
