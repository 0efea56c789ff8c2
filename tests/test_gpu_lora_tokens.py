"""A token's adapter result does not depend on the other requests of the batch: neither their
sizes nor what is not finite in them change its bits."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


class Batch:
    """Tokens of two adapters in turn; every fifth is loud.  Enough of them for tiles."""

    def __init__(self, T, r, dtype, quiet):
        gen = torch.Generator().manual_seed(T + r)
        K, N = 1024, 512
        self.T, self.K, self.N, self.r = T, K, N, r
        rnd = lambda *s, std=1.0: (torch.randn(s, generator=gen) * std).to(DEV, dtype)  # noqa
        self.loud = torch.arange(T, device=DEV) % 5 == 0
        size = torch.where(self.loud, 2e4, quiet).unsqueeze(1)
        self.x = (torch.randn((T, K), generator=gen).clamp(-3, 3).to(DEV) * size).to(dtype)
        self.dy = (torch.randn((T, N), generator=gen).clamp(-3, 3).to(DEV) * size).to(dtype)
        self.a, self.b = rnd(2, r, K, std=K ** -0.5), rnd(2, N, r, std=0.05)
        self.ids = torch.arange(T, device=DEV) % 2
        self.base = torch.zeros((T, N), dtype=dtype, device=DEV)
        self.s = 64.0


@pytest.mark.parametrize("dtype,quiet", [(F16, 1e-4), (F16, 4e-6), (BF16, 1e-12)])
@pytest.mark.parametrize("T,r", [(2000, 16), (3000, 20), (2000, 40), (2500, 100)])
def test_sizes_of_others(T, r, dtype, quiet):
    o = Batch(T, r, dtype, quiet)
    announce(f"sizes of others {T} {r} {dtype} {quiet}")
    out = mmfp4.lora_add(o.base, o.x, o.a, o.b, o.ids, o.s)
    dx = mmfp4.lora_backward(o.dy, o.x, o.a, o.b, o.ids, o.s)[0]
    q = ~o.loud
    pick = lambda w, t: w.double()[o.ids[t]]                               # noqa: E731
    few = torch.nonzero(q).flatten()[:200]
    A, B = pick(o.a, few), pick(o.b, few)
    for got, v, first, second in ((out, o.x, A, B),
                                  (dx, o.dy, B.transpose(1, 2), A.transpose(1, 2))):
        v = v[few].double().unsqueeze(2)
        ref = o.s * torch.bmm(second, torch.bmm(first, v)).squeeze(2)
        terms = o.s * torch.bmm(second.abs(), torch.bmm(first.abs(), v.abs())).squeeze(2)
        # half a step of the result, 16 bits of H or 22, fp32 sums; the smallest numbers
        half, bits = torch.finfo(dtype).eps / 2, 2.0 ** (-16 if dtype == BF16 else -21)
        tol = half * ref.abs() + (bits + 2 * (v.shape[1] + r) * 2.0 ** -24) * terms
        tol += torch.finfo(dtype).smallest_normal * half
        assert ((got[few].double() - ref).abs() <= tol).all()
    # the same tokens beside others of their own size
    o.x[o.loud] = (o.x[o.loud].float() / 2e4 * quiet).to(dtype)
    o.dy[o.loud] = (o.dy[o.loud].float() / 2e4 * quiet).to(dtype)
    again = mmfp4.lora_add(o.base, o.x, o.a, o.b, o.ids, o.s)
    assert torch.equal(out[q], again[q])
    assert torch.equal(dx[q], mmfp4.lora_backward(o.dy, o.x, o.a, o.b, o.ids, o.s)[0][q])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_what_is_not_finite_in_others(dtype, bad):
    o = Batch(2000, 16, dtype, 1.0)
    want = mmfp4.lora_add(o.base, o.x, o.a, o.b, o.ids, o.s)
    dx = mmfp4.lora_backward(o.dy, o.x, o.a, o.b, o.ids, o.s)[0]
    o.x[o.loud, 3], o.dy[o.loud, 5] = bad, bad
    q = ~o.loud
    assert torch.equal(mmfp4.lora_add(o.base, o.x, o.a, o.b, o.ids, o.s)[q], want[q])
    assert torch.equal(mmfp4.lora_backward(o.dy, o.x, o.a, o.b, o.ids, o.s)[0][q], dx[q])
