"""The MXFP4 product and its input gradient on every tile, with their contraction whole and split, and
the experts' block where one expert has most rows."""

from __future__ import annotations

import pytest
import torch

import mmfp4
import mx_plan
from gpu_helpers import DEV, announce
from mmfp4 import _lib
from mx_reference import check, half_step, quantize, rounded, sum_error, values
from test_gpu_moe_mxfp4 import case as moe_case
from test_gpu_moe_route import compare

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# (tile, whether K is split): rows, columns, K
PRODUCTS = {
    (0, False): (515, 14340, 800), (0, True): (1030, 4099, 14368),
    (1, False): (1030, 4099, 800), (1, True): (200, 8201, 14368),
    (2, False): (200, 8201, 800), (2, True): (65, 4099, 14368),
    (3, False): (77, 8201, 1056), (3, True): (130, 2050, 8224),
    (4, False): (77, 75, 1056), (4, True): (65, 75, 8224)}
# (tile, whether N is split, whether dY is fp32): rows, N, K
GRADIENTS = {
    (0, False, False): (515, 500, 8224), (0, True, False): (200, 4099, 2080),
    (1, False, False): (515, 500, 4128), (1, True, False): (515, 4099, 544),
    (2, False, False): (333, 500, 544), (2, True, False): (40, 8201, 1056),
    (0, False, True): (515, 500, 8224), (0, True, True): (200, 2050, 2080),
    (1, False, True): (515, 500, 4128), (1, True, True): (515, 2050, 544),
    (2, False, True): (515, 500, 1056), (2, True, True): (40, 4099, 544)}


def normal(*shape, dtype=torch.float32, std=1.0, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def test_these_sizes_take_these_tiles():
    """The number of splits shows in the workspace that the library asks for."""
    lib = _lib.load()
    pitch = lambda n: (n + 3) // 4 * 16                                     # noqa: E731
    for (tile, split), (M, N, K) in PRODUCTS.items():
        t, splits = mx_plan.product(M, N, K)
        assert (t, splits > 1) == (tile, split), (M, N, K, t, splits)
        units, kp = -(-K // 256), (K + 511) // 512 * 512
        scales = units * 2048 * (-(-M // 256) + -(-N // 256))
        sums = splits * pitch(M * N) if split else 0
        assert lib.mm_mxfp4_gemm_workspace_bytes(M, N, K) == 65536 + M * kp // 2 + scales + sums
    for (tile, split, fp32), (M, N, K) in GRADIENTS.items():
        t, splits = mx_plan.gradient(M, N, K, fp32)
        assert (t, splits > 1) == (tile, split), (M, N, K, t, splits)
        pad = 0 if K % 128 == 0 else (N * ((K // 32 + 3) // 4 * 4) + 255) // 256 * 256
        sums = splits * pitch(M * K) if split else 0
        want = 65536 + pad + sums if pad + sums else 0
        for type_ in (0,) if fp32 else (1, 2):
            assert lib.mm_mxfp4_gemm_backward_workspace_bytes(M, N, K, type_) == want


def near(out, ref, terms):
    """fp32 sums of `terms` products, eight or more of them at a time: each addition is off by 2^-23 of
    a partial sum at most if it cuts off, by half of that on average, and partial sums of numbers of
    both signs are smaller than the whole."""
    assert float((out.double() - ref).norm() / ref.norm()) < terms / 8 * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("tile,split", PRODUCTS)
def test_product(tile, split):
    M, N, K = PRODUCTS[tile, split]
    w, s = quantize(normal(N, K, std=0.02, seed=2))
    rw = values(w, s)
    for dtype in TYPES:
        announce(f"mxfp4_gemm tile {tile} split {split} {dtype}")
        x = normal(M, K, dtype=dtype, seed=1)
        rx = rounded(x)
        ref = rx @ rw.t()
        y = mmfp4.mxfp4_gemm(x, w, s, torch.float32)
        near(y, ref, K)
        sums = sum_error(rx.abs() @ rw.abs().t(), K // 64 + 16)
        check(y, ref, (sums + half_step(ref, torch.float32)) * (1 + 2.0 ** -8))
        assert torch.equal(mmfp4.mxfp4_gemm(x, w, s), y.to(dtype))          # the sums, rounded once


@pytest.mark.gpu
@pytest.mark.parametrize("tile,split,fp32", GRADIENTS)
def test_gradient(tile, split, fp32):
    M, N, K = GRADIENTS[tile, split, fp32]
    w, s = quantize(normal(N, K, std=0.02, seed=2))
    s[N // 2:N // 2 + 70, ::3] = 100            # stages of fp16 gradients that take two terms
    rw = values(w, s)
    for dtype in TYPES[:1] if fp32 else TYPES[1:]:
        announce(f"mxfp4_gemm_backward tile {tile} split {split} {dtype}")
        dy = normal(M, N, dtype=dtype, seed=1)
        ref = dy.double() @ rw
        dx = mmfp4.mxfp4_gemm_backward(dy, w, s, torch.float32)
        terms = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dtype]
        near(dx, ref, terms * N)
        sums = sum_error(dy.double().abs() @ rw.abs(), terms * N // 4 + 40)
        check(dx, ref, (sums + half_step(ref, torch.float32)) * (1 + 2.0 ** -8))
        assert torch.equal(mmfp4.mxfp4_gemm_backward(dy, w, s), dx.to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [9, 100, 700])
def test_every_bit_of_a_gradient_counts(m):
    """Gradients whose leading 8 bits are alike: what is left of them is all of the result."""
    announce(f"mxfp4_gemm_backward low bits {m}")
    w, s = quantize(normal(1000, 640, std=0.02, seed=3))
    for scale in (None, 100):
        if scale is not None:
            s[::90, ::2] = scale
        rw = values(w, s)
        for dtype, low in ((torch.float16, 10), (torch.float32, 23)):
            g = torch.Generator(DEV).manual_seed(m)
            bits = torch.randint(0, 1 << (low - 7), (m, 1000), generator=g, device=DEV)
            dy = (1 + bits.double() * 2.0 ** -low).to(dtype)
            ref = dy.double() @ rw
            dx = mmfp4.mxfp4_gemm_backward(dy, w, s, torch.float32).double()
            lead = rw.sum(0)                    # what the leading bits alone give
            terms = 2 if dtype == torch.float16 else 3
            err = sum_error(dy.double().abs() @ rw.abs(), terms * 1000 // 4 + 40)
            check(dx, ref, err * (1 + 2.0 ** -8))
            if dtype == torch.float16:
                # the low bits are 2^-9 of the whole, the sums' error some 2^-20 of it
                assert float((dx - ref).norm()) < 0.01 * float((ref - lead).norm())


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,H,I,ids", [
    (511, 1, 128, 512, 256, 7), (300, 2, 200, 288, 96, 199), (2000, 1, 1024, 64, 32, 0)])
def test_experts_with_most_rows(T, k, E, H, I, ids):
    """On average less than 4 rows an expert, so that the weights are streamed, and nearly all of
    them one expert's: sixteen at a time."""
    announce(f"moe_mlp_mxfp4 one expert {T} {k} {E}")
    g = torch.Generator(DEV).manual_seed(T)
    which = torch.randint(-1, E, (T, k), generator=g, device=DEV)
    which = torch.where(torch.rand((T, k), generator=g, device=DEV) < 0.95, ids, which)
    moe_case(T, k, E, H, I, torch.bfloat16, ids=which)


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,H,I", [(5, 3, 8, 96, 160), (40, 8, 128, 2048, 768), (300, 4, 8, 1024, 544)])
def test_experts_round_once(T, k, E, H, I):
    """What an expert gives a token stays fp32: a 16-bit result is the fp32 one, rounded."""
    announce(f"moe_mlp_mxfp4 one rounding {T}")
    gu, dn = quantize(normal(E, 2 * I, H, std=0.02)), quantize(normal(E, H, I, std=0.02, seed=1))
    probs, ids = torch.topk(torch.softmax(normal(T, E, std=1.5, seed=2), 1), k)
    for dtype in (torch.float16, torch.bfloat16):
        x = normal(T, H, dtype=dtype, seed=3)
        whole = mmfp4.moe_mlp_mxfp4(x.float(), *gu, *dn, ids, probs)
        assert torch.equal(mmfp4.moe_mlp_mxfp4(x, *gu, *dn, ids, probs), whole.to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("E,groups,keep,k", [(256, 1, 1, 20), (64, 1, 1, 33), (128, 8, 4, 17),
                                             (256, 16, 16, 64), (60, 4, 4, 16)])
def test_routing_of_more_experts_than_lanes(E, groups, keep, k, renorm):
    """Sixteen lanes share a token; each keeps one chosen expert at a time."""
    announce(f"moe_route {E} k {k} {renorm}")
    for softmax in (False, True):
        logits = normal(2100, E, std=1.5, seed=E + k)
        compare(logits, k, softmax, normal(E, std=0.05, seed=1), groups, keep, renorm, 2.5)
