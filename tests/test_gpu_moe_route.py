"""Routing with sigmoid or softmax scores, bias and groups, and its gradient, against the
definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import mmfp4
from gpu_helpers import DEV, announce
from mx_reference import half_step, route, route_grad

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(*shape, dtype=torch.float32, std=1.0, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def compare(logits, k, softmax=False, bias=None, groups=1, keep=1, renorm=True, scale=1.0):
    w, ids = mmfp4.moe_route(logits, k, scoring="softmax" if softmax else "sigmoid", bias=bias,
                             num_groups=groups, topk_groups=keep, renormalize=renorm, scale=scale)
    rw, rids = route(logits, k, softmax, bias, groups, keep, renorm, scale)
    assert w.dtype == torch.float32 and ids.dtype == torch.int64
    assert torch.equal(ids, rids)
    # computed in 64 bits, rounded once; `scale` reaches the kernel as an fp32 number
    bound = half_step(rw, torch.float32) * (1 + 2.0 ** -20) + rw.abs() * 2.0 ** -24
    bad = ~((w.double() - rw).abs() <= bound) & ~(torch.isnan(w) & torch.isnan(rw))
    assert not bad.any()
    return w, ids


@pytest.mark.parametrize("T", [1, 3, 33, 2500])
@pytest.mark.parametrize("E,groups,keep,k", [
    (8, 1, 1, 2), (16, 4, 2, 3), (64, 1, 1, 6), (60, 4, 3, 8), (128, 8, 4, 8), (256, 8, 4, 8),
    (160, 16, 5, 10), (257, 1, 1, 20), (480, 8, 3, 8), (512, 64, 10, 64), (1024, 1, 1, 1),
    (1000, 20, 20, 33), (5, 5, 5, 5), (1, 1, 1, 1), (7, 7, 2, 2)])
def test_route(T, E, groups, keep, k):
    announce(f"moe_route {T} x {E} groups {keep}/{groups} k {k}")
    i = T + E + k
    logits = normal(T, E, dtype=TYPES[i % 3], std=1.5, seed=i)
    bias = normal(E, std=0.05, seed=i + 1) if i % 2 else None
    compare(logits, k, i % 4 < 2, bias, groups, keep, i % 5 != 0, 2.5 if i % 7 < 3 else 1.0)


@pytest.mark.parametrize("T", [4, 3000])
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("groups,keep", [(1, 1), (8, 3)])
def test_ties_go_to_the_lower_index(softmax, groups, keep, T):
    announce(f"moe_route ties {softmax} {groups} {T}")
    g = torch.Generator(DEV).manual_seed(5)
    logits = torch.randint(-2, 3, (T, 64), generator=g, device=DEV).to(torch.bfloat16)
    logits[0] = 0
    compare(logits, 8, softmax, None, groups, keep)
    compare(logits, 8, softmax, torch.zeros(64, device=DEV), groups, keep)


@pytest.mark.parametrize("T", [6, 2100])
@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
def test_masks_and_ends(softmax, groups, keep, T):
    announce(f"moe_route masks {softmax} {groups} {T}")
    logits = normal(T, 32, std=1.0, seed=9)
    logits[0] = -math.inf                                # nothing left
    logits[1, 3:] = -math.inf                            # fewer than k left
    logits[2, ::2] = torch.finfo(torch.float32).min
    logits[3, 5] = 200.0
    logits[4] = -200.0
    w, ids = compare(logits, 4, softmax, None, groups, keep)
    assert torch.equal(w[0], torch.zeros(4, device=DEV))
    compare(logits, 4, softmax, normal(32, std=0.1), groups, keep)
    # a bias of -inf closes an expert
    bias = torch.zeros(32, device=DEV)
    bias[[0, 9, 31]] = -math.inf
    _, ids = mmfp4.moe_route(logits[2:], 4, scoring="softmax" if softmax else "sigmoid", bias=bias,
                             num_groups=groups, topk_groups=keep)
    assert not torch.isin(ids, torch.tensor([0, 9, 31], device=DEV)).any()


@pytest.mark.parametrize("softmax", [False, True])
def test_nan_and_infinity(softmax):
    announce(f"moe_route nan {softmax}")
    logits = normal(5, 64, seed=2)
    logits[0, 7] = math.nan
    logits[1] = math.nan
    logits[2, 9] = math.inf
    for groups, keep in ((1, 1), (8, 2)):
        w, ids = mmfp4.moe_route(logits, 6, scoring="softmax" if softmax else "sigmoid",
                                 num_groups=groups, topk_groups=keep)
        assert int(ids.min()) >= 0 and int(ids.max()) < 64
        assert all(len(set(r)) == 6 for r in ids.tolist())
        assert torch.isfinite(w[3:]).all()
        if softmax:
            assert torch.isnan(w[:3]).all()
        else:
            assert torch.isfinite(w[0]).all() and 7 not in ids[0].tolist()
            assert torch.isnan(w[1]).all()
            # (1 and a small second score may lose to two middling ones where groups compete)
            assert groups > 1 or int(ids[2, 0]) == 9


@pytest.mark.parametrize("T", [1, 5, 2300])
@pytest.mark.parametrize("E,k", [(8, 2), (60, 4), (128, 8), (256, 20), (500, 8), (1024, 64)])
def test_gradient(T, E, k):
    i = T + E + k
    softmax, renorm, dtype = i % 2 == 0, i % 3 != 0, TYPES[i % 3]
    announce(f"moe_route_backward {T} x {E} k {k} {softmax} {renorm} {dtype}")
    logits = normal(T, E, dtype=dtype, std=1.5, seed=i)
    dw = normal(T, k, std=1e-2, seed=i + 1)
    _, ids = mmfp4.moe_route(logits, k, scoring="softmax" if softmax else "sigmoid")
    dl = mmfp4.moe_route_backward(dw, logits, ids, scoring="softmax" if softmax else "sigmoid",
                                  renormalize=renorm, scale=2.5)
    ref = route_grad(dw, logits, ids, softmax, renorm, 2.5)
    assert dl.dtype == dtype
    # 64 bits, rounded once; what two terms cancel is lost of 64 bits
    bound = half_step(ref, dtype) * (1 + 2.0 ** -20) + 1e-15
    assert ((dl.double() - ref).abs() <= bound).all()


def test_gradient_of_repeated_and_foreign_ids():
    announce("moe_route_backward repeated ids")
    for T in (3, 2200):
        logits = normal(T, 40, seed=4)
        dw = normal(T, 20, seed=5)
        g = torch.Generator(DEV).manual_seed(6)
        ids = torch.randint(-3, 43, (T, 20), generator=g, device=DEV)
        for softmax in (False, True):
            for renorm in (False, True):
                dl = mmfp4.moe_route_backward(dw, logits, ids, renormalize=renorm,
                                              scoring="softmax" if softmax else "sigmoid")
                ref = route_grad(dw, logits, ids, softmax, renorm)
                bound = half_step(ref, torch.float32) * (1 + 2.0 ** -20) + 1e-14
                assert ((dl.double() - ref).abs() <= bound).all()


def test_gradient_of_ids_beyond_32_bits():
    """An id whose low 32 bits name an expert is foreign all the same."""
    announce("moe_route_backward large ids")
    for T in (3, 2200):
        logits, dw = normal(T, 40, seed=4), normal(T, 4, seed=5)
        ids = torch.tensor([3, 2 ** 32 + 3, 7, -2 ** 40 + 7], device=DEV).expand(T, 4)
        want = mmfp4.moe_route_backward(dw, logits, torch.where(ids < 40, ids, -1).clamp(min=-1))
        assert torch.equal(mmfp4.moe_route_backward(dw, logits, ids), want)
        ref = route_grad(dw, logits, ids, False, True)
        bound = half_step(ref, torch.float32) * (1 + 2.0 ** -20) + 1e-14
        assert ((want.double() - ref).abs() <= bound).all()


def test_autograd_and_differences():
    announce("moe_route autograd")
    logits = normal(7, 48, seed=8)
    for scoring in ("sigmoid", "softmax"):
        leaf = logits.clone().requires_grad_(True)
        w, ids = mmfp4.moe_route(leaf, 5, scoring=scoring, num_groups=6, topk_groups=3, scale=2.0,
                                 bias=normal(48, std=0.02))
        assert w.requires_grad and not ids.requires_grad
        c = normal(7, 5, seed=9)
        (w * c).sum().backward()
        # differences of the definition in 64 bits, along a direction, the choice held
        d = normal(7, 48, seed=10).double()

        def value(step):
            l = logits.double() + step * d
            s = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, 1)
            u = s.gather(1, ids)
            return float((2.0 * u / u.sum(1, keepdim=True) * c.double()).sum())
        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        got = float((leaf.grad.double() * d).sum())
        # the differences' own error: step^2 and 64-bit rounding over the step
        assert abs(got - slope) <= 1e-6 * float((leaf.grad.double() * d).abs().sum()) + 1e-9
        with pytest.raises(RuntimeError):
            w2, _ = mmfp4.moe_route(leaf, 5, scoring=scoring)
            grad, = torch.autograd.grad(w2.sum(), leaf, create_graph=True)
            grad.sum().backward()


def test_operands():
    announce("moe_route operands")
    logits = normal(2, 3, 64, dtype=torch.float16)
    w, ids = mmfp4.moe_route(logits, 4)
    assert w.shape == ids.shape == (2, 3, 4)
    f, i = mmfp4.moe_route(logits.view(6, 64), 4)
    assert torch.equal(w.view(6, 4), f) and torch.equal(ids.view(6, 4), i)
    wide = torch.zeros(6, 100, dtype=torch.float16, device=DEV)
    wide[:, 30:94] = logits.view(6, 64)
    w2, i2 = mmfp4.moe_route(wide[:, 30:94], 4)
    assert torch.equal(w2, f) and torch.equal(i2, i)
    w2, i2 = mmfp4.moe_route(logits.view(6, 64).t().contiguous().t(), 4,
                             bias=torch.zeros(64, dtype=torch.bfloat16, device=DEV))
    assert torch.equal(w2, f) and torch.equal(i2, i)
    dl = mmfp4.moe_route_backward(w.half(), logits, ids.int())
    assert dl.shape == logits.shape and dl.dtype == torch.float16
    assert torch.equal(dl, mmfp4.moe_route_backward(w.half().float(), logits, ids))
    w0, i0 = mmfp4.moe_route(logits[:0], 4)
    assert w0.shape == i0.shape == (0, 3, 4)
    assert mmfp4.moe_route_backward(w0, logits[:0], i0).shape == (0, 3, 64)
