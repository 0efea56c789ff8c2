"""The experts' block on MXFP4 weights against its definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import mmfp4
from gpu_helpers import DEV, announce
from mx_reference import half_step, quantize, rounded, sum_error, values

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(*shape, dtype=torch.float32, std=1.0, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def weights(E, H, I, seed=1):
    return (*quantize(normal(E, 2 * I, H, std=0.02, seed=seed)),
            *quantize(normal(E, H, I, std=0.02, seed=seed + 1)))


def reference(x, gu, gus, dn, dns, ids, probs):
    """(out, bound) in 64 bits.  silu(g) * u comes to the kernel with an error of fp32 sums; a
    value that lies that near the middle between two codes may round either way, and a block
    whose largest lies that near a power of two may take either scale: `loose` is what that can
    move.  The rest are the sums' and the two roundings' errors."""
    T, H = x.shape
    k, E = ids.shape[1], gu.shape[0]
    I = 8 * dn.shape[2]
    rx = rounded(x)
    out = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    for e in range(E):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        wg, wd = values(gu[e], gus[e]), values(dn[e], dns[e])
        both = rx[t] @ wg.t()
        mags = rx[t].abs() @ wg.abs().t()
        g, u = both.chunk(2, 1)
        dg, du = sum_error(mags, H // 64 + 16).chunk(2, 1)
        sig = torch.sigmoid(g)
        h = g * sig * u
        # |d silu| <= 1.1 |dg|; the kernel's own exp, quotient and products: 2^-20 of the value
        # and of |g| times it (an error of the exponent's argument)
        err = 1.1 * dg * (u.abs() + du) + (g * sig).abs() * du + h.abs() * (1 + g.abs()) * 2.0 ** -20
        words, scales = quantize(h)
        a = values(words, scales)
        lo, hi = rounded(h - err), rounded(h + err)
        move = torch.maximum((a - lo).abs(), (a - hi).abs())
        # the scale: if a bound of the block's largest magnitude crosses a power of two, all its
        # values may move by half of the coarser step, which is a sixth of the largest at most
        top = h.abs().unflatten(1, (-1, 32))
        er = err.unflatten(1, (-1, 32))
        _, e0 = torch.frexp((top - er).clamp_min(0).amax(-1))
        _, e1 = torch.frexp((top + er).amax(-1))
        cross = (e0 != e1).unsqueeze(-1).expand(-1, -1, 32).flatten(1)
        big = top.amax(-1, keepdim=True).expand(-1, -1, 32).flatten(1)
        move = torch.where(cross, torch.maximum(move, big / 3), move)
        y = a @ wd.t()
        dy = move @ wd.abs().t() + sum_error((a.abs() + move) @ wd.abs().t(), I // 64 + 16)
        dy += half_step(y.abs() + dy, x.dtype)
        p = probs[t, j].double().unsqueeze(1)
        out.index_add_(0, t, p * y)
        bound.index_add_(0, t, p.abs() * (dy * (1 + 2.0 ** -10) + (y.abs() + dy) * (k + 1) * 2.0 ** -24))
    return out, bound * (1 + 2.0 ** -10) + half_step(out.abs() + bound, x.dtype)


def case(T, k, E, H, I, dtype=torch.bfloat16, ids=None, seed=0, int32=False):
    x = normal(T, H, dtype=dtype, seed=seed)
    w = weights(E, H, I, seed=seed + 1)
    logits = normal(T, E, std=1.5, seed=seed + 3)
    probs, own = torch.topk(torch.softmax(logits, 1), k)
    ids = own if ids is None else ids
    ids = ids.int() if int32 else ids
    y = mmfp4.moe_mlp_mxfp4(x, *w, ids, probs)
    assert y.dtype == dtype and y.shape == (T, H)
    ref, bound = reference(x, *w, ids, probs)
    off = (y.double() - ref).abs() - bound
    assert float(off.max()) <= 0, f"beyond its bound by {float(off.max()):.3g}"
    # the bound's loose part is rare: most values are as near as their type allows
    tight = half_step(ref, dtype) + 4 * half_step(ref.abs().amax(1, keepdim=True), dtype) + \
        2.0 ** -17 * ref.abs().amax(1, keepdim=True)
    assert float(((y.double() - ref).abs() > tight).double().mean()) < 0.05
    return x, w, ids, probs, y


@pytest.mark.parametrize("T,k,E,H,I", [
    (1, 1, 1, 32, 32), (1, 2, 8, 256, 128), (5, 3, 8, 96, 160), (17, 8, 16, 512, 768),
    (40, 8, 128, 2048, 768), (130, 2, 4, 288, 96), (300, 4, 8, 1024, 544), (64, 6, 60, 640, 352),
    (1000, 8, 16, 2048, 768), (33, 1, 1, 4128, 64), (2, 2, 300, 64, 64)])
def test_moe_mlp(T, k, E, H, I):
    announce(f"moe_mlp_mxfp4 T {T} k {k} E {E} H {H} I {I}")
    case(T, k, E, H, I, TYPES[(T + H) % 3], seed=T, int32=T % 2 == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [4, 200])
def test_types(T, dtype):
    announce(f"moe_mlp_mxfp4 {T} {dtype}")
    case(T, 4, 8, 256, 256, dtype)


@pytest.mark.parametrize("T", [9, 400])
def test_uneven_repeated_and_foreign_ids(T):
    """All tokens to one expert, one expert twice, ids outside the experts', tokens without any."""
    announce(f"moe_mlp_mxfp4 ids {T}")
    g = torch.Generator(DEV).manual_seed(3)
    ids = torch.randint(-2, 10, (T, 4), generator=g, device=DEV)
    ids[0] = 5
    ids[1] = -1
    ids[2] = 99
    x, w, ids, probs, y = case(T, 4, 8, 256, 96, ids=ids)
    assert not y[1].any() and not y[2].any()
    case(T, 4, 8, 256, 96, ids=torch.full((T, 4), 7, device=DEV))
    case(T, 4, 8, 256, 96, ids=torch.full((T, 4), -5, device=DEV))


def test_tokens_do_not_depend_on_others():
    announce("moe_mlp_mxfp4 others")
    for T in (12, 500):
        x, w, ids, probs, y = case(T, 2, 4, 256, 128, torch.float16)
        other = x.clone()
        other[::2] = math.inf
        z = mmfp4.moe_mlp_mxfp4(other, *w, ids, probs)
        assert torch.equal(z[1::2], y[1::2])
        assert torch.isnan(z[::2]).all()
        again = mmfp4.moe_mlp_mxfp4(x, *w, ids, probs)
        assert torch.equal(again, y)


def test_operands_and_refusals():
    announce("moe_mlp_mxfp4 operands")
    x, w, ids, probs, y = case(20, 2, 4, 256, 128, torch.bfloat16)
    wide = torch.zeros(20, 512, dtype=torch.bfloat16, device=DEV)
    wide[:, 100:356] = x
    assert torch.equal(mmfp4.moe_mlp_mxfp4(wide[:, 100:356], *w, ids, probs), y)
    both = torch.stack([ids, ids], 2)[..., 0]
    assert torch.equal(mmfp4.moe_mlp_mxfp4(x, *w, both, probs.double()), y)
    assert mmfp4.moe_mlp_mxfp4(x[:0], *w, ids[:0], probs[:0]).shape == (0, 256)
    bad = [(x[:, :64], *w, ids, probs), (x, *w, ids[:3], probs), (x, *w, ids, probs[:, :1]),
           (x, w[0], w[1], w[2][:, :64], w[3][:, :64], ids, probs),
           (x, w[0][:3], w[1][:3], w[2], w[3], ids, probs)]
    for args in bad:
        with pytest.raises(ValueError):
            mmfp4.moe_mlp_mxfp4(*args)
    with pytest.raises(TypeError):
        mmfp4.moe_mlp_mxfp4(x, *w, ids.float(), probs)


def test_routed_experts_together():
    """Routing, quantization, the experts' block and a projection of its result, as a layer uses
    them: every step from what the one before returned."""
    announce("moe layer mxfp4")
    T, E, H, I, k = 50, 16, 512, 256, 4
    x = normal(T, H, dtype=torch.bfloat16, seed=1)
    gate = normal(E, H, std=H ** -0.5, seed=2, dtype=torch.bfloat16)
    gu, gus = mmfp4.mxfp4_quantize(normal(E, 2 * I, H, std=0.02, seed=3))
    dn, dns = mmfp4.mxfp4_quantize(normal(E, H, I, std=0.02, seed=4))
    pw, ps = mmfp4.mxfp4_quantize(normal(192, H, std=0.02, seed=5))
    probs, ids = mmfp4.moe_route(x @ gate.t(), k, bias=normal(E, std=0.01, seed=6), num_groups=4,
                                 topk_groups=2, scale=2.5)
    y = mmfp4.moe_mlp_mxfp4(x, gu, gus, dn, dns, ids, probs)
    ref, bound = reference(x, gu, gus, dn, dns, ids, probs)
    assert ((y.double() - ref).abs() <= bound).all()
    z = mmfp4.mxfp4_gemm(y, pw, ps)
    rz = rounded(y) @ values(pw, ps).t()
    lim = sum_error(rounded(y).abs() @ values(pw, ps).abs().t(), 32) + half_step(rz, z.dtype)
    assert ((z.double() - rz).abs() <= lim * (1 + 2.0 ** -8)).all()
