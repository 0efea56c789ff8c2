"""MXFP4 and routing from their definitions, in 64 bits (torch, any device)."""

from __future__ import annotations

import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
MIDS = (GRID[1:] + GRID[:-1]) / 2


def block_exponents(x: torch.Tensor) -> torch.Tensor:
    """[*, K] -> int64 [*, K/32]: the powers of two, from the largest magnitudes' fp64 bits."""
    top = x.double().unflatten(-1, (-1, 32)).abs().amax(-1)
    _, e = torch.frexp(top)                              # top = f * 2^e, f in [0.5, 1)
    return torch.where(top > 0, e.long() - 3, -127).clamp_min(-127)


def quantize(x: torch.Tensor):
    """Words int32 [*, K/8] and scales uint8 [*, K/32] of finite x."""
    e = block_exponents(x)
    v = x.double().unflatten(-1, (-1, 32)) / torch.exp2(e.double()).unsqueeze(-1)
    a, mids = v.abs(), MIDS.to(x.device)
    code = torch.bucketize(a, mids)                      # a tie stays at the lower code
    tie = (code < 7) & (a == mids[code.clamp_max(6)])
    code = code + (tie & (code % 2 == 1)) + 8 * torch.signbit(v)
    code = code.flatten(-2).unflatten(-1, (-1, 8))
    words = (code << (4 * torch.arange(8, device=x.device))).sum(-1)
    words = torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)
    return words, (e + 127).to(torch.uint8)


def values(words: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp64 [*, K]; a block with scale 255 is NaN."""
    code = (words.long().unsqueeze(-1) >> (4 * torch.arange(8, device=words.device))) & 15
    v = GRID.to(words.device)[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, math.nan, s)
    return (v.flatten(-2).unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def rounded(x: torch.Tensor) -> torch.Tensor:
    return values(*quantize(x))


def half_step(ref: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Half a step of `dtype` at ref: relative to the value, or of its smallest subnormal."""
    info = torch.finfo(dtype)
    return ref.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def sum_error(terms_abs_sum: torch.Tensor, adds: int) -> torch.Tensor:
    """What `adds` fp32 additions in any order may lose of a sum: each is off by at most 2^-24
    of a partial sum, which the terms' magnitudes bound."""
    return terms_abs_sum * (adds * 2.0 ** -24)


def check(out: torch.Tensor, ref: torch.Tensor, bound: torch.Tensor, what: str = "") -> None:
    out = out.double()
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(out), nan), f"{what}: NaNs elsewhere"
    off = torch.where(nan, 0.0, (out - ref).abs() - bound)
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, f"{what}: beyond its bound by {worst:.3g} at {int(off.argmax())}"


def route(logits, k, softmax=False, bias=None, groups=1, keep=1, renorm=True, scale=1.0):
    """(weights fp64 [T, k], ids int64 [T, k]) token by token, from the definition."""
    T, E = logits.shape
    n = E // groups
    l = logits.double().cpu()
    if softmax:
        s = torch.softmax(l, 1)
        s[(l == -math.inf).all(1)] = 0.0
    else:
        s = torch.sigmoid(l)
    c = s + (0 if bias is None else bias.double().cpu())
    c = torch.where(torch.isnan(c), -math.inf, c)
    ids = torch.empty(T, k, dtype=torch.int64)
    for t in range(T):
        row = c[t].tolist()
        tops = []
        for g in range(groups):
            best = sorted(row[g * n:(g + 1) * n], reverse=True)[:2]
            tops.append(sum(best))
        kept = sorted(range(groups), key=lambda g: (-tops[g], g))[:keep]
        free = [e for g in kept for e in range(g * n, (g + 1) * n)]
        ids[t] = torch.tensor(sorted(free, key=lambda e: (-row[e], e))[:k])
    w = s.gather(1, ids)
    if renorm:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return (w * scale).to(logits.device), ids.to(logits.device)


def route_grad(dw, logits, ids, softmax=False, renorm=True, scale=1.0):
    """dlogits fp64 by torch's own differentiation of the weights."""
    leaf = logits.double().detach().requires_grad_(True)
    s = torch.softmax(leaf, 1) if softmax else torch.sigmoid(leaf)
    live = (ids >= 0) & (ids < logits.shape[1])
    w = torch.where(live, s.gather(1, ids.clamp(0, logits.shape[1] - 1)), 0.0)
    if renorm:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    (w * scale * dw.double()).sum().backward()
    return leaf.grad
