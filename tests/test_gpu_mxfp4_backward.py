"""The input gradient of the MXFP4 product against its definition in 64 bits."""

from __future__ import annotations

import math

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


def weight(n, k, seed=1):
    return quantize(normal(n, k, std=0.02, seed=seed))


def bound_of(dy, rw, ref, dtype):
    # every product is exact; fp16 is two terms and fp32 three, each one more set of additions
    terms = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dy.dtype]
    mags = dy.double().abs() @ rw.abs()
    return (sum_error(mags, terms * dy.shape[1] // 4 + 40) + half_step(ref, dtype)) * (1 + 2.0 ** -8)


def case(m, n, k, dtype, out_dtype=None, seed=0):
    dy = normal(m, n, dtype=dtype, std=1e-3, seed=seed)
    w, s = weight(n, k, seed=seed + 1)
    rw = values(w, s)
    ref = dy.double() @ rw
    dx = mmfp4.mxfp4_gemm_backward(dy, w, s) if out_dtype is None else \
        mmfp4.mxfp4_gemm_backward(dy, w, s, out_dtype)
    assert dx.dtype == (out_dtype or dtype)
    check(dx, ref, bound_of(dy, rw, ref, dx.dtype), f"{m} x {n} x {k}")
    if dx.dtype == torch.float32:      # far nearer than the bound on average
        off = (dx.double() - ref).norm() / ref.norm()
        assert float(off) < 1e-6 if dtype == torch.float32 else 2e-6


@pytest.mark.parametrize("m", [1, 2, 31, 32, 33, 64, 100, 129, 257, 515])
@pytest.mark.parametrize("n,k", [(64, 256), (33, 32), (264, 992), (1, 96), (500, 4096), (4099, 160)])
def test_backward(m, n, k):
    announce(f"mxfp4_gemm_backward {m} x {n} x {k}")
    case(m, n, k, TYPES[(m + n) % 3], seed=m)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("m", [3, 200])
def test_types(m, dtype, out_dtype):
    announce(f"mxfp4_gemm_backward {m} {dtype} -> {out_dtype}")
    case(m, 136, 640, dtype, out_dtype)


@pytest.mark.parametrize("m,n,k,dtype", [
    (8, 14336, 4096, torch.float16), (509, 4096, 4096, torch.float16),
    (2048, 14336, 4096, torch.bfloat16), (4099, 1000, 4128, torch.float32),
    (1030, 72, 14336, torch.bfloat16)])
def test_large(m, n, k, dtype):
    announce(f"mxfp4_gemm_backward {m} x {n} x {k}")
    case(m, n, k, dtype)


@pytest.mark.parametrize("n", list(range(1, 70)))
def test_every_tail(n):
    announce(f"mxfp4_gemm_backward n={n}")
    case(5, n, 64, TYPES[n % 3], seed=n)
    case(70, n, 160, TYPES[(n + 1) % 3], seed=n)


@pytest.mark.parametrize("dtype", TYPES)
def test_range(dtype):
    """Scales and gradients at the ends of their ranges enter exactly."""
    announce(f"mxfp4_gemm_backward range {dtype}")
    info = torch.finfo(dtype)
    for m in (20, 140):
        dy = torch.zeros(m, 64, dtype=dtype, device=DEV)
        dy[torch.arange(m), torch.arange(m) % 64] = normal(m, dtype=dtype)
        dy[0, 0], dy[1, 1], dy[2, 2] = info.max, -info.max, info.tiny
        w, s = weight(64, 96)
        s[:, 0] = torch.arange(64, device=DEV) % 8           # the smallest scales
        s[:, 1] = 127
        ref = dy.double() @ values(w, s)
        dx = mmfp4.mxfp4_gemm_backward(dy, w, s, torch.float32)
        # one product each: exact but for fp32's ends and a split's lowest bits beside zeros
        big = ref.abs() > torch.finfo(torch.float32).max
        assert torch.equal(torch.isinf(dx), big)
        lim = half_step(ref, torch.float32) * 3 + 2.0 ** -126
        off = torch.where(big, 0.0, (dx.double() - ref).abs() - lim)
        assert float(off.max()) <= 0


@pytest.mark.parametrize("m", [7, 150])
def test_fp16_exponents(m):
    """fp16 gradients down to the subnormal ones, and weights whose scales leave fp16's range in some
    rows and columns only: each product is exact however a stage takes them."""
    announce(f"mxfp4_gemm_backward fp16 exponents m={m}")
    dy = normal(m, 640, dtype=torch.float16)
    dy = torch.ldexp(dy.float(), -(torch.arange(640, device=DEV) % 24).float()).half()
    w, s = weight(640, 512)
    s[64:128, 3] = 113                       # one stage of one column tile
    s[300, :] = 141
    s[450:460, 9:] = 90
    s[500:600, :8] = 0                       # zeros under the least scale
    w[500:600, :32] = 0
    rw = values(w, s)
    ref = dy.double() @ rw
    dx = mmfp4.mxfp4_gemm_backward(dy, w, s, torch.float32)
    check(dx, ref, bound_of(dy, rw, ref, torch.float32), f"m={m}")
    tiny = torch.full((m, 640), 2.0 ** -24, dtype=torch.float16, device=DEV)     # the smallest one
    one = torch.full_like(s, 127)
    ref = tiny.double() @ values(w, one)
    dx = mmfp4.mxfp4_gemm_backward(tiny, w, one, torch.float32)
    assert torch.equal(dx.double(), ref)     # sums of multiples of 2^-25 below 2^-12: exact


@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite(dtype):
    announce(f"mxfp4_gemm_backward not finite {dtype}")
    for m in (8, 140):
        dy = normal(m, 72, dtype=dtype)
        dy[1, 3], dy[2, 70] = math.nan, math.inf
        w, s = weight(72, 96)
        w[70] = 0x22222222                                    # ones: inf times them is inf
        dx = mmfp4.mxfp4_gemm_backward(dy, w, s)
        assert torch.isnan(dx[1]).all() and torch.isinf(dx[2]).all()
        keep = [i for i in range(m) if i not in (1, 2)]
        assert torch.isfinite(dx[keep]).all()
        s[5, 1] = 255
        dx = mmfp4.mxfp4_gemm_backward(dy, w, s)[keep]
        assert torch.isnan(dx[:, 32:64]).all() and torch.isfinite(dx[:, :32]).all()
        assert torch.isfinite(dx[:, 64:]).all()


def test_operands():
    announce("mxfp4_gemm_backward operands")
    w, s = weight(96, 512)
    dy = normal(2, 3, 5, 96, dtype=torch.bfloat16)
    dx = mmfp4.mxfp4_gemm_backward(dy, w, s)
    assert dx.shape == (2, 3, 5, 512)
    flat = dx.view(30, 512)
    wide = torch.zeros(30, 200, dtype=torch.bfloat16, device=DEV)
    wide[:, 33:129] = dy.view(30, 96)
    assert torch.equal(mmfp4.mxfp4_gemm_backward(wide[:, 33:129], w, s), flat)
    assert torch.equal(mmfp4.mxfp4_gemm_backward(dy.view(30, 96).t().contiguous().t(), w, s), flat)
    stacked, scales = torch.cat([w, w]), torch.cat([s, s])
    assert torch.equal(mmfp4.mxfp4_gemm_backward(dy, stacked[96:], scales[96:]), dx)
    assert mmfp4.mxfp4_gemm_backward(dy[:0], w, s).shape == (0, 3, 5, 512)
    assert not mmfp4.mxfp4_gemm_backward(dy[..., :0], w[:0], s[:0]).any()
    with pytest.raises(ValueError):
        mmfp4.mxfp4_gemm_backward(dy[..., :64], w, s)
    with pytest.raises(TypeError):
        mmfp4.mxfp4_gemm_backward(dy.int(), w, s)


def test_autograd_is_straight_through():
    announce("mxfp4 autograd")
    w, s = weight(80, 256)
    for dtype in TYPES:
        x = normal(3, 7, 256, dtype=dtype).requires_grad_(True)
        c = normal(3, 7, 80, dtype=dtype, seed=5)
        y = mmfp4.mxfp4_gemm(x, w, s)
        assert torch.equal(y, mmfp4.mxfp4_gemm(x.detach(), w, s))
        y.backward(c)
        assert torch.equal(x.grad, mmfp4.mxfp4_gemm_backward(c, w, s))
        # of the formula: differences of c . (x W^T), which the product is but for x's rounding
        d = normal(3, 7, 256, seed=6).double()
        rw = values(w, s)
        slope = float((c.double() * (d @ rw.t())).sum())
        got = float((x.grad.double() * d).sum())
        lim = (half_step(x.grad.double(), dtype) * d.abs()).sum() * 1.01 + \
            sum_error((c.double().abs() @ rw.abs() * d.abs()).sum(), 100)
        assert abs(got - slope) <= float(lim)
    with pytest.raises(RuntimeError):
        x = normal(2, 256).requires_grad_(True)
        g, = torch.autograd.grad(mmfp4.mxfp4_gemm(x, w, s).sum(), x, create_graph=True)
        g.sum().backward()


def test_layer_and_adapters():
    announce("MXFP4Linear")
    lin = torch.nn.Linear(256, 96).to(DEV)
    layer = mmfp4.MXFP4Linear.from_linear(lin)
    words, scales = mmfp4.mxfp4_quantize(lin.weight.detach())
    assert torch.equal(layer.packed_weights, words) and torch.equal(layer.scales, scales)
    for dtype in TYPES:
        x = normal(4, 9, 256, dtype=dtype)
        y = layer(x)
        assert y.dtype == dtype and y.shape == (4, 9, 96)
        assert torch.equal(y, mmfp4.mxfp4_gemm(x, words, scales) + lin.bias.detach().to(dtype))
        leaf = x.clone().requires_grad_(True)
        layer(leaf).sum().backward()
        assert torch.equal(leaf.grad, layer.input_grad(torch.ones_like(y)))
    layer.bias.requires_grad_(True)
    layer(x).float().sum().backward()
    assert torch.equal(layer.bias.grad, torch.full((96,), 36.0, device=DEV))
    state = layer.state_dict()
    other = mmfp4.MXFP4Linear(torch.zeros_like(words), torch.zeros_like(scales), lin.bias.detach())
    other.load_state_dict(state)
    assert torch.equal(other(x), layer(x))
    both = mmfp4.LoRALinear(other, rank=4, num_adapters=3, dtype=torch.bfloat16)
    torch.nn.init.normal_(both.lora_b, std=0.1)
    ids = torch.arange(36, device=DEV) % 4 - 1
    x = normal(36, 256, dtype=torch.bfloat16).requires_grad_(True)
    z = both(x, ids)
    ref = mmfp4.lora_add(other(x.detach()), x.detach(), both.lora_a.detach(),
                         both.lora_b.detach(), ids)
    assert torch.equal(z, ref)
    c = normal(36, 96, dtype=torch.bfloat16, seed=3)
    z.backward(c)
    dx, da, db = mmfp4.lora_backward(c, x.detach(), both.lora_a.detach(), both.lora_b.detach(),
                                     ids, dx_base=other.input_grad(c))
    assert torch.equal(x.grad, dx) and torch.equal(both.lora_a.grad, da)
    assert torch.equal(both.lora_b.grad, db)


def test_training_step_of_a_quantized_block():
    """Forward and backward of two layers as a training step runs them, against 64 bits step by
    step from what the step before gave."""
    announce("mxfp4 training step")
    w1, w2 = weight(320, 256, seed=1), weight(64, 320, seed=2)
    x = normal(50, 256, dtype=torch.bfloat16).requires_grad_(True)
    h = mmfp4.mxfp4_gemm(x, *w1)
    a = torch.relu(h)
    y = mmfp4.mxfp4_gemm(a, *w2)
    c = normal(50, 64, dtype=torch.bfloat16, seed=4)
    y.backward(c)
    da = mmfp4.mxfp4_gemm_backward(c, *w2)
    dh = da * (h > 0)
    assert torch.equal(x.grad, mmfp4.mxfp4_gemm_backward(dh, *w1))
    ref = rounded(a) @ values(*w2).t()
    lim = sum_error(rounded(a).abs() @ values(*w2).abs().t(), 32) + half_step(ref, y.dtype)
    assert ((y.double() - ref).abs() <= lim * (1 + 2.0 ** -8)).all()
