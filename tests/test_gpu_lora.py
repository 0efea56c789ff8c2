"""Low-rank adapters of many requests and their gradients, against the formulas in 64 bits.

Tolerances are error bounds, element by element.  A sum of n terms in fp32 is off by at most
n * 2^-23 of the terms' magnitudes.  Where the tokens go by tiles, h and dh reach the second
product in two parts of the operands' type: off by 2^-16 (bf16: 2^-9 * 2^-9, and the first
part's error is measured against a rounded one) or less, and by 2^-38 of the tile's largest
value.  The result is off by half a step of its type."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def half_step(t):
    return torch.finfo(t).eps / 2


class Case:
    def __init__(self, T, K, N, r, L, dtype, seed=0, ids=None, x_scale=1.0):
        gen = torch.Generator().manual_seed(1000 * seed + T + K + N + r + L)
        rnd = lambda *s, std=1.0: (torch.randn(s, generator=gen) * std).to(DEV, dtype)  # noqa
        self.T, self.K, self.N, self.r, self.L, self.dtype = T, K, N, r, L, dtype
        self.x, self.base = rnd(T, K, std=x_scale), rnd(T, N)
        self.a, self.b = rnd(L, r, K, std=K ** -0.5), rnd(L, N, r, std=0.1)
        self.dy, self.dx_base = rnd(T, N, std=1e-2), rnd(T, K, std=1e-2)
        self.s = (0.5 + torch.rand(L, generator=gen)).to(DEV)
        if ids is None:
            ids = torch.randint(-1, L + 1, (T,), generator=gen)   # L: out of range too
        self.ids = ids.to(DEV)

    def per_token(self):
        """One-hot over adapters times nothing: rows of tokens without an adapter are zero."""
        e = torch.arange(self.L, device=DEV)
        return (self.ids.view(-1, 1) == e).double()

    def down(self, v, w):
        """(s v w^T, the same of magnitudes) [T, r]; w [L, r, C]."""
        m = self.per_token() * self.s.double()
        h = torch.einsum("tc,lrc->tlr", v.double(), w.double())
        a = torch.einsum("tc,lrc->tlr", v.double().abs(), w.double().abs())
        return (h * m.unsqueeze(2)).sum(1), (a * m.unsqueeze(2)).sum(1)

    def up(self, h, w):
        """h w of each token's adapter; w [L, r, C]."""
        m = self.per_token()
        return torch.einsum("tl,tr,lrc->tc", m, h, w.double())

    def grad(self, h, v):
        """[L, r, C]: sum over tokens of h^T v."""
        return torch.einsum("tl,tr,tc->lrc", self.per_token(), h, v.double())

    def h_error(self, h, mags, width):
        return width * 2.0 ** -23 * mags + 2.0 ** -16 * h.abs() + 2.0 ** -38 * h.abs().max()


def check(out, ref, carried, dtype, what):
    assert out.dtype == dtype and out.shape == ref.shape, (what, out.dtype, out.shape)
    tiny = torch.finfo(dtype).smallest_normal * half_step(dtype)
    tol = half_step(dtype) * (1 + 1e-3) * ref.abs() + tiny + (1 + half_step(dtype)) * carried
    off = (out.double() - ref).abs()
    # a value that rounds past the type's largest, 65504 + 16 of fp16, is infinite (h = 1e7
    # times 70 gradients of 1e-2 gives a db of 7e4)
    edge = torch.finfo(dtype).max * (1 + half_step(dtype) / 2)
    over = out.isinf() & (out.sign() == ref.sign()) & (ref.abs() + tol >= edge)
    bad = ~((off <= tol) | over)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst " \
        f"{float((off / tol).max())} of the bound"


def check_add(c, out, dtype=None, base=None):
    bt = c.b.transpose(1, 2)
    h, mags = c.down(c.x, c.a)
    base = (c.base if base is None else base).double()
    d, dm = c.up(h, bt), c.up(h.abs(), bt.abs())
    err = c.up(c.h_error(h, mags, c.K + 8), bt.abs()) + (2 * c.r + 8) * 2.0 ** -23 * \
        (dm + base.abs())
    check(out, base + d, err, dtype or c.dtype, "out")


def check_backward(c, got, with_base=True):
    dx, da, db = got
    bt = c.b.transpose(1, 2)
    h, hm = c.down(c.x, c.a)
    dh, dm = c.down(c.dy, bt)
    eh, ed = c.h_error(h, hm, c.K + 8), c.h_error(dh, dm, c.N + 8)
    base = c.dx_base.double() if with_base else torch.zeros_like(c.x, dtype=torch.float64)
    check(dx, base + c.up(dh, c.a),
          c.up(ed, c.a.abs()) + (2 * c.r + 8) * 2.0 ** -23 * (c.up(dh.abs(), c.a.abs()) +
                                                             base.abs()), c.dtype, "dx")
    n = (2 * c.T + 64) * 2.0 ** -23
    check(da, c.grad(dh, c.x),
          c.grad(ed, c.x.abs()) + n * c.grad(dh.abs(), c.x.abs()), c.dtype, "da")
    check(db, c.grad(h, c.dy).transpose(1, 2),
          (c.grad(eh, c.dy.abs()) + n * c.grad(h.abs(), c.dy.abs())).transpose(1, 2), c.dtype,
          "db")


SIZES = [  # T, K, N, r, L
    (1, 64, 64, 16, 1), (1, 4096, 512, 16, 8), (2, 8, 8, 1, 3), (5, 72, 40, 4, 3),
    (7, 100, 33, 5, 2), (32, 512, 257, 64, 32), (63, 264, 1000, 12, 70), (64, 136, 64, 130, 4),
    (65, 64, 64, 16, 1), (65, 520, 100, 8, 4), (100, 33, 1, 3, 5), (130, 1, 65, 17, 2),
    (257, 2048, 264, 33, 3), (300, 200, 515, 64, 9), (500, 776, 320, 100, 2),
    (1111, 328, 136, 16, 100), (900, 64, 72, 200, 1), (2100, 512, 256, 16, 1),
    # forward by tiles (many tokens per adapter, wide factors)
    (300, 4096, 515, 40, 2), (1111, 2048, 264, 64, 3), (700, 1000, 1030, 130, 2),
    (400, 2056, 1001, 33, 4), (1500, 4000, 96, 16, 1), (260, 64, 8200, 24, 1),
    (9000, 256, 200, 64, 3),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,K,N,r,L", SIZES)
def test_add(T, K, N, r, L, dtype):
    announce(f"lora_add {T} {K} {N} {r} {L} {dtype}")
    c = Case(T, K, N, r, L, dtype)
    out = mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s)
    check_add(c, out)
    none = (c.ids < 0) | (c.ids >= L)
    assert torch.equal(out[none], c.base[none])
    assert torch.equal(out, mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids.to(torch.int32), c.s))
    mine = c.base.clone()
    assert mmfp4.lora_add(mine, c.x, c.a, c.b, c.ids, c.s, out=mine) is mine
    assert torch.equal(mine, out)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,K,N,r,L", SIZES)
def test_backward(T, K, N, r, L, dtype):
    announce(f"lora_backward {T} {K} {N} {r} {L} {dtype}")
    c = Case(T, K, N, r, L, dtype)
    got = mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s, dx_base=c.dx_base)
    check_backward(c, got)
    again = mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s)
    check_backward(c, again, with_base=False)
    assert torch.equal(again[1], got[1]) and torch.equal(again[2], got[2])
    for e in range(L):
        if not (c.ids == e).any():
            assert not got[1][e].any() and not got[2][e].any()


@pytest.mark.parametrize("T", [3, 200])
def test_one_adapter_without_ids(T):
    c = Case(T, 136, 72, 8, 1, F16, ids=torch.zeros(T, dtype=torch.int64))
    a, b = c.a[0], c.b[0]
    c.s[0] = 0.5
    out = mmfp4.lora_add(c.base, c.x, a, b, scaling=0.5)
    check_add(c, out)
    assert torch.equal(out, mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, torch.tensor(0.5).cuda()))
    dx, da, db = mmfp4.lora_backward(c.dy, c.x, a, b, scaling=0.5, dx_base=c.dx_base)
    assert da.shape == a.shape and db.shape == b.shape
    check_backward(c, (dx, da[None], db[None]))


@pytest.mark.parametrize("T", [4, 100])
def test_tokens_without_adapters(T):
    """A batch in which no token has an adapter: outputs are the bases, gradients zeros."""
    c = Case(T, 64, 72, 8, 3, BF16, ids=torch.full((T,), -1))
    assert torch.equal(mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s), c.base)
    dx, da, db = mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s, dx_base=c.dx_base)
    assert torch.equal(dx, c.dx_base) and not da.any() and not db.any()
    assert not mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s)[0].any()


@pytest.mark.parametrize("T", [4, 100])
def test_fp16_base_of_bf16_tokens(T):
    """The products return fp16 whatever their input: base fp16, everything else bf16."""
    c = Case(T, 256, 72, 8, 3, BF16)
    base = torch.randn((T, 72), device=DEV).half()
    out = mmfp4.lora_add(base, c.x, c.a, c.b, c.ids, c.s)
    check_add(c, out, BF16, base)


@pytest.mark.parametrize("T", [6, 200])
@pytest.mark.parametrize("mag", [1e-6, 1e4])
def test_sizes_of_h(T, mag):
    """h far above and below fp16's range of full precision (h reaches 1e6 and 1e-6)."""
    c = Case(T, 512, 64, 16, 2, F16, x_scale=min(mag, 1e3))
    c.b *= 1e-2
    if mag > 1e3:
        c.s *= 1e3
        c.b *= 1e-2
    check_add(c, mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s))
    c.dy *= mag if mag < 1 else 1.0
    check_backward(c, mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s, dx_base=c.dx_base))


@pytest.mark.parametrize("T", [5, 90])
def test_non_finite_tokens_stay_by_themselves(T):
    c = Case(T, 64, 72, 8, 2, F16)
    ref = mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s)
    c.ids[2] = 0
    c.x[2, 3] = float("nan")
    out = mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s)
    keep = [i for i in range(T) if i != 2]
    if T > 64:      # a tile's power of two goes by its largest value: equal within the bound
        assert out[keep].isfinite().all()
    else:
        assert torch.equal(out[keep], ref[keep])
    assert out[2].isnan().all()
    c.ids[2] = -1                                   # without an adapter x is not looked at
    out = mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s)
    assert out.isfinite().all()


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_non_finite_tokens_leave_the_others_their_bits(bad):
    """Small H beside an infinite one in the same tile: 1e-5 would be a subnormal of fp16."""
    c = Case(4200, 64, 72, 8, 1, F16, x_scale=1e-5, ids=torch.zeros(4200, dtype=torch.int64))
    c.b *= 100
    c.base.zero_()
    clean = mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s)
    row = c.x[5].clone()
    c.x[5, 3] = bad
    out = mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s)
    assert not out[5].isfinite().any()
    c.x[5], out[5] = row, clean[5]
    check_add(c, out)


def test_fp32_base_of_dx_stays_fp32():
    """What reaches an fp32 x through the projection does not pass through fp16."""
    c = Case(70, 64, 48, 8, 2, F32)
    dx, da, db = mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s)
    small = c.dx_base * 1e-9
    got = mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s, dx_base=small)
    assert got[0].dtype == F32 and torch.equal(got[0], dx + small)
    assert torch.equal(got[1], da) and torch.equal(got[2], db)
    none = (c.ids < 0) | (c.ids >= 2)
    assert none.any() and torch.equal(got[0][none], small[none])


def test_forms_of_the_operands():
    """Leading axes, strides, odd offsets, factors of another type, fp32 tokens, no tokens."""
    c = Case(12, 64, 72, 8, 3, F16)
    ref = mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s)
    lead = mmfp4.lora_add(c.base.view(3, 4, 72), c.x.view(3, 4, 64), c.a, c.b, c.ids.view(3, 4),
                          c.s)
    assert lead.shape == (3, 4, 72) and torch.equal(lead.view(12, 72), ref)
    wide = torch.zeros((12, 101), dtype=F16, device=DEV)
    wide[:, 5:69] = c.x
    off = torch.empty(12 * 72 + 1, dtype=F16, device=DEV)[1:].view(12, 72)
    off.copy_(c.base)
    assert torch.equal(mmfp4.lora_add(off, wide[:, 5:69], c.a, c.b, c.ids, c.s), ref)
    f32 = mmfp4.lora_add(c.base, c.x.float(), c.a.float(), c.b.float(), c.ids, c.s)
    assert f32.dtype == F16 and torch.equal(f32, ref)
    g = mmfp4.lora_backward(c.dy, c.x, c.a.float(), c.b.float(), c.ids, c.s)
    assert g[0].dtype == F16 and g[1].dtype == F32 and g[2].dtype == F32
    half = mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s)
    assert torch.equal(g[1].half(), half[1]) and torch.equal(g[2].half(), half[2])
    empty = mmfp4.lora_add(c.base[:0], c.x[:0], c.a, c.b, c.ids[:0], c.s)
    assert empty.shape == (0, 72)
    g = mmfp4.lora_backward(c.dy[:0], c.x[:0], c.a, c.b, c.ids[:0], c.s)
    assert g[0].shape == (0, 64) and not g[1].any() and not g[2].any()


def test_out_beside_the_operands():
    """out may be base itself; anything else that shares its memory is refused."""
    gen = torch.Generator().manual_seed(31)
    T, K = 6, 64
    a, b = (torch.randn((1, *s), generator=gen).to(DEV, F16) for s in ((4, K), (K, 4)))
    both = torch.randn((T + 1, K), generator=gen).to(DEV, F16)
    x, base = both[:T], torch.randn((T, K), generator=gen).to(DEV, F16)
    for name, out, bs in (("x", x, base), ("x", both[1:], base), ("base", both[1:], both[:T])):
        with pytest.raises(ValueError, match=f"memory with {name}"):
            mmfp4.lora_add(bs, x if name == "x" else base, a, b, out=out)
    want = mmfp4.lora_add(base, x, a, b)
    assert torch.equal(mmfp4.lora_add(base, x, a, b, out=base), want)
    # columns of one tensor are not contiguous as `out`, but may be base and x
    wide = torch.randn((T, 2 * K), generator=gen).to(DEV, F16)
    want = mmfp4.lora_add(wide[:, :K].contiguous(), wide[:, K:].contiguous(), a, b)
    assert torch.equal(mmfp4.lora_add(wide[:, :K], wide[:, K:], a, b, out=base), want)


def test_gradients_by_differences():
    """da, db and dx against central differences of the sum in 64 bits."""
    c = Case(70, 24, 16, 3, 2, F16)
    dx, da, db = mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s)

    def loss(x, a, b):
        m = c.per_token() * c.s.double()
        return torch.einsum("tl,tk,lrk,lnr,tn->", m, x, a, b, c.dy.double())
    p = [t.double() for t in (c.x, c.a, c.b)]
    rng = torch.Generator().manual_seed(1)
    for which, got in ((0, dx), (1, da), (2, db)):
        d = torch.randn(p[which].shape, generator=rng, dtype=torch.float64).to(DEV)
        hi, lo = ([q + s * 1e-4 * d if i == which else q for i, q in enumerate(p)]
                  for s in (1, -1))
        num = float((loss(*hi) - loss(*lo)) / 2e-4)
        terms = float((got.double() * d).abs().sum())
        assert abs(float((got.double() * d).sum()) - num) <= 2.0 ** -10 * terms


@pytest.mark.parametrize("T,K", [(4, 256), (150, 256), (500, 4096)])
def test_capture(T, K):
    """Captured once, replayed on new tokens, ids and factors with eager work between; two
    graphs in turn."""
    c = Case(T, K, 200, 16, 4, BF16)

    def step():
        out = mmfp4.lora_add(c.base, c.x, c.a, c.b, c.ids, c.s)
        return (out, *mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s, dx_base=c.dx_base))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    with torch.cuda.stream(side):
        step()
        for g in graphs:
            with torch.cuda.graph(g, stream=side):
                held.append(step())
    torch.cuda.current_stream().wait_stream(side)
    gen = torch.Generator().manual_seed(3)
    for i in range(4):
        for t in (c.x, c.a, c.b, c.dy, c.base):
            t.copy_(torch.randn(t.shape, generator=gen))
        c.ids.copy_(torch.randint(-1, 4, (T,), generator=gen))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for outs in held:
            for a, b in zip(outs, step()):
                assert torch.equal(a, b), i


def test_beside_the_projections():
    """lora_add after the framework's own products, as a layer runs them."""
    K, N, g = 256, 128, 64
    gen = torch.Generator().manual_seed(4)
    w = (torch.randn((N, K), generator=gen) * 0.05).half().to(DEV)
    words, scales = mmfp4.quantize_fp4(w, group_size=g)
    for T in (3, 80):
        c = Case(T, K, N, 8, 3, F16)
        base = mmfp4.marlin_gemm_fp4(c.x, words, scales, g)
        check_add(c, mmfp4.lora_add(base, c.x, c.a, c.b, c.ids, c.s), F16, base)
        dxb = mmfp4.marlin_gemm_fp4_backward(c.dy, words, scales, g)
        c.dx_base = dxb
        check_backward(c, mmfp4.lora_backward(c.dy, c.x, c.a, c.b, c.ids, c.s, dx_base=dxb))
