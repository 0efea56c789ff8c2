"""Gradients at the ends of their types' ranges: rows are carried in fp16 under a power of two
each."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
K, N, G = 256, 320, 64
# a row's largest magnitude: the subnormals' end, both sides of 2^-110 and of 2^126, the last
SIZES = (2.0 ** -149, 3 * 2.0 ** -149, 2.0 ** -141, 2.0 ** -133, 1.5 * 2.0 ** -130, 2.0 ** -111,
         2.0 ** -109, 1.0, 2.0 ** 100, 2.0 ** 125, 1.5 * 2.0 ** 126, 1.75 * 2.0 ** 127)


def weights(gen):
    w = (torch.randn((N, K), generator=gen) * 0.02).half().to(DEV)
    words, scales = mmfp4.quantize_fp4(w, group_size=G)
    return words, scales, mmfp4.dequant_fp4(words, scales, K, N, G).double()


def rows(gen, M, dtype):
    """Three values a row, the largest of each of SIZES and neighbours down to 2^-30 of it."""
    dy = torch.zeros((M, N), dtype=torch.float64)
    for i in range(M):
        at = torch.randperm(N, generator=gen)[:3]
        sign = torch.randint(0, 2, (3,), generator=gen) * 2.0 - 1
        dy[i, at] = SIZES[i % len(SIZES)] * sign.double() * torch.tensor(
            [1.0, 0.3, 2.0 ** -(i % 31)], dtype=torch.float64)
    return dy.to(dtype).to(DEV)


def bound(dy, ref, terms, dtype):
    """Half a step of the result (or of the smallest number), fp32 carried in 11 bits, and what
    lies 2^-40 below a row's largest; fp32 sums are exact to 2^-22 here."""
    carried = 2.0 ** -11 if dy.dtype == F32 else 0
    low = dy.double().abs().amax(1, keepdim=True) * 2.0 ** -40 * N
    smallest = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return torch.finfo(dtype).eps / 2 * ref.abs() + (carried + 2.0 ** -22) * terms + low + smallest


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [12, 48, 600])
def test_products(M, dtype):
    gen = torch.Generator().manual_seed(1)
    words, scales, W = weights(gen)
    dy = rows(gen, M, dtype)
    ref, terms = dy.double() @ W.t(), dy.double().abs() @ W.abs().t()
    assert ref.abs().max() < torch.finfo(dtype).max
    announce(f"range {M} {dtype}")
    q = mmfp4.mmfp4_fused_qkv_backward(dy, dy * 0, dy * 0, *(words, scales) * 3, G)
    for dx in (mmfp4.marlin_gemm_fp4_backward(dy, words, scales, G), q):
        assert ((dx.double() - ref).abs() <= bound(dy, ref, terms, dtype)).all()
        assert dx[SIZES.index(2.0 ** 100)].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gated_block(dtype):
    """dg and du of 11 bits each; u = 1 and g = 1 leave dh its size."""
    gen = torch.Generator().manual_seed(2)
    words, scales, W = weights(gen)
    dh = rows(gen, 60, dtype) / 4
    gu = torch.ones((60, 2 * N), dtype=F16, device=DEV)
    sig = torch.sigmoid(torch.ones((), dtype=torch.float64, device=DEV))
    ref = (dh.double() * sig * (2 - sig)) @ W.t() + (dh.double() * sig) @ W.t()
    terms = 2 * dh.double().abs() @ W.abs().t()
    dx = mmfp4.fused_gate_up_swiglu_backward(dh, gu, words, scales, words, scales, G)
    tol = bound(dh, ref, terms, dtype) + 2.0 ** -10 * terms + 2 * 2.0 ** -149
    assert ((dx.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [4, 48])
def test_an_infinity_leaves_the_others(M, dtype):
    """Finite values beside an infinity do not become infinite themselves: the result is that of
    the formula, infinite or NaN."""
    gen = torch.Generator().manual_seed(3)
    words, scales, W = weights(gen)
    dy = torch.zeros((M, N), dtype=dtype, device=DEV)
    dy[0, 7], dy[0, 9:40] = float("inf"), 1e6
    dy[1, 3], dy[1, 9:40] = -float("inf"), -1e30
    dy[2, 9:40] = 1e6
    dy[3, 5], dy[3, 50:60] = float("nan"), 1e6
    ref = dy.double() @ W.t()
    dx = mmfp4.marlin_gemm_fp4_backward(dy, words, scales, G).double()
    assert torch.equal(dx.isnan(), ref.isnan()) and ref[0].isinf().any()
    assert torch.equal(dx.isinf(), ref.isinf())
    assert torch.equal(dx[:2][ref[:2].isinf()], ref[:2][ref[:2].isinf()])
    assert ((dx[2] - ref[2]).abs() <= 2.0 ** -8 * (dy[2].double() @ W.abs().t())).all()
