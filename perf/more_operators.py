"""The operators on microscaled 4-bit floating point (MXFP4: E2M1 codes, one power of two per
block of 32 along K), the routing to experts, and what is measured of them.  A case is a dict of
plain values; its "path" says what runs:

  quantize    rows of activations or weights to MXFP4 codes and scales, and back to values
  gemm        x . W^T with both sides MXFP4: x is quantized in the call, W is kept quantized
  gemm_bwd    the gradient of that product's input, straight through x's rounding: dy . W
  route       scores, balance bias, groups, top-k and weights of every token's experts
  route_step  that, and the gradient of the logits
  moe         the experts' gated feed-forward block on MXFP4 weights, for routed tokens

Blocks follow the OCP microscaling format: a block's scale is 2^(floor(log2(its largest
magnitude)) - 2), at least 2^-127, and its values are rounded to nearest, ties to even, and
saturate at 6.  Weights are N(0, 0.02) quantized so; activations N(0, 1), with a few channels
ten times as large, as trained models have them; gradients N(0, 1e-3).  Inside the experts'
block silu(gate) * up is quantized again, from its 32-bit value.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0,
        -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-20         # added to the sum that weights are divided by


def listed():
    # hidden 4096, intermediate 14336: the benchmark's dense model; 128 experts of 2048 -> 768,
    # 8 per token: its mixture of experts
    return [
        # a short prompt's activations, in 32 bits as a norm leaves them
        {"name": "quantize_t65", "path": "quantize", "type": "fp32", "rows": 65, "k": 2048},
        # a whole weight as it is converted
        {"name": "quantize_weight", "path": "quantize", "type": "bf16", "rows": 14336, "k": 4096},
        # one token, where latency counts
        {"name": "gemm_m1", "path": "gemm", "type": "bf16", "m": 1, "n": 4096, "k": 4096},
        # a decode batch through the widest layer
        {"name": "gemm_m24", "path": "gemm", "type": "fp16", "m": 24, "n": 14336, "k": 4096},
        # a short prompt, odd in rows and columns
        {"name": "gemm_m333", "path": "gemm", "type": "bf16", "m": 333, "n": 4099, "k": 14336},
        # a long prompt
        {"name": "gemm_m2048", "path": "gemm", "type": "bf16", "m": 2048, "n": 14336, "k": 4096},
        # training beside frozen weights: an odd number of tokens, fp16 gradients
        {"name": "gemm_bwd_m509", "path": "gemm_bwd", "type": "fp16", "m": 509, "n": 4096,
         "k": 4096},
        # a full batch through the widest layer
        {"name": "gemm_bwd_m2048", "path": "gemm_bwd", "type": "bf16", "m": 2048, "n": 14336,
         "k": 4096},
        # a decode batch routed with a balance bias and groups
        {"name": "route_t32", "path": "route", "type": "bf16", "tokens": 32, "experts": 256,
         "top_k": 8, "scoring": "sigmoid", "bias": True, "groups": 8, "topk_groups": 4,
         "renormalize": True, "scale": 2.5},
        # a training batch, softmax over all experts
        {"name": "route_step_t4096", "path": "route_step", "type": "fp32", "tokens": 4096,
         "experts": 128, "top_k": 8, "scoring": "softmax", "bias": False, "groups": 1,
         "topk_groups": 1, "renormalize": True, "scale": 1.0},
        # a decode batch through all experts
        {"name": "moe_t32", "path": "moe", "type": "fp16", "tokens": 32, "experts": 128,
         "top_k": 8, "hidden": 2048, "inter": 768},
        # a prompt
        {"name": "moe_t1000", "path": "moe", "type": "bf16", "tokens": 1000, "experts": 128,
         "top_k": 8, "hidden": 2048, "inter": 768},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(("quantize", "quantize", "gemm", "gemm", "gemm", "gemm", "gemm_bwd",
                       "gemm_bwd", "route", "route_step", "moe", "moe"))
    case = {"path": path, "type": rng.choice(("fp16", "bf16", "bf16", "fp32"))}
    if path == "quantize":
        k = 32 * _log(rng, 4, 448)
        return {**case, "rows": min(_log(rng, 1, 16384), 58_000_000 // k), "k": k}
    if path in ("gemm", "gemm_bwd"):
        k, n = 32 * _log(rng, 8, 448), 8 * _log(rng, 32, 1792) + rng.choice((0, 0, 0, 4, 1))
        most = 120_000_000_000 if path == "gemm" else 60_000_000_000
        return {**case, "m": min(_log(rng, 1, 8192), most // (n * k)), "n": n, "k": k}
    if path in ("route", "route_step"):
        groups = rng.choice((1, 1, 4, 8))
        experts = groups * rng.choice((8, 16, 24, 32, 60))
        keep = rng.randint((groups + 1) // 2, groups)
        top_k = rng.choice((1, 2, 4, 6, 8))
        return {**case, "tokens": min(_log(rng, 1, 16384), 4_000_000 // experts),
                "experts": experts, "top_k": top_k,
                "scoring": rng.choice(("sigmoid", "softmax")), "bias": rng.random() < 0.6,
                "groups": groups, "topk_groups": keep,
                "renormalize": top_k > 1 and rng.random() < 0.7, "scale": rng.choice((1.0, 2.5))}
    hidden, inter = 32 * _log(rng, 16, 128), 32 * _log(rng, 8, 64)
    experts = rng.choice((8, 16, 64, 128))
    experts = min(experts, 600_000_000 // (3 * hidden * inter))
    top_k = min(experts, rng.choice((1, 2, 4, 8)))
    tokens = min(_log(rng, 1, 4096), 38_000_000_000 // (3 * hidden * inter * top_k))
    return {**case, "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden,
            "inter": inter}


# ------------------------------------------------------------------- inputs
class _Inputs:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.gen = torch.Generator(self.dev).manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=self.gen, device=self.dev) * std).to(dtype)

    def tokens(self, t, k, dtype):
        """Activations: one channel in a hundred is ten times as large."""
        big = torch.rand(k, generator=self.gen, device=self.dev) < 0.01
        return (self.normal(t, k) * (1.0 + 9.0 * big)).to(dtype)

    def weight(self, *shape):
        """A quantized weight: words [*, K/8] of E2M1 codes, low nibble first, and scales
        [*, K/32], the biased exponents of the blocks' powers of two."""
        w = self.normal(*shape, std=0.02).unflatten(-1, (-1, 32))
        _, e = torch.frexp(w.abs().amax(-1))
        e = (e - 3).clamp_min(-127)
        v = torch.ldexp(w, -e.unsqueeze(-1))
        mids = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device=self.dev)
        codes = torch.bucketize(v.abs(), mids, out_int32=True) + 8 * (v < 0)
        shift = 4 * torch.arange(8, device=self.dev, dtype=torch.int32)
        words = torch.sum(codes.unflatten(-1, (4, 8)) << shift, dim=-1, dtype=torch.int32)
        return words.flatten(-2).contiguous(), (e + 127).to(torch.uint8)


def prepare(case, seed):
    make, dt, path = _Inputs(seed), TYPES[case["type"]], case["path"]
    st = {"path": path}
    if path == "quantize":
        return {**st, "x": make.tokens(case["rows"], case["k"], dt)}
    if path == "gemm":
        return {**st, "w": make.weight(case["n"], case["k"]),
                "x": make.tokens(case["m"], case["k"], dt)}
    if path == "gemm_bwd":
        return {**st, "w": make.weight(case["n"], case["k"]),
                "dy": make.normal(case["m"], case["n"], std=1e-3, dtype=dt)}
    if path in ("route", "route_step"):
        t, e = case["tokens"], case["experts"]
        st["logits"] = make.normal(t, e, std=1.5, dtype=dt)
        st["bias"] = make.normal(e, std=0.05) if case["bias"] else None
        st["how"] = {v: case[v] for v in ("top_k", "scoring", "groups", "topk_groups",
                                          "renormalize", "scale")}
        if path == "route_step":
            st["dw"] = make.normal(t, case["top_k"], std=1e-2)
        return st
    t, e, h, i, k = (case[v] for v in ("tokens", "experts", "hidden", "inter", "top_k"))
    scores = torch.softmax(make.normal(t, e, std=1.5), -1)
    probs, ids = torch.topk(scores, k)
    rows = int(torch.bincount(ids.flatten(), minlength=e).max())     # of the busiest expert
    return {**st, "x": make.tokens(t, h, dt), "gate_up": make.weight(e, 2 * i, h),
            "down": make.weight(e, h, i), "ids": ids,
            "probs": probs / probs.sum(-1, keepdim=True), "rows": rows}


# ---------------------------------------------------------------- plain form
def _plain_rounded(x):
    """The MXFP4 values of x [*, K], in 32 bits."""
    v = x.float().unflatten(-1, (-1, 32))
    _, e = torch.frexp(v.abs().amax(-1, keepdim=True))
    e = (e - 3).clamp_min(-127)
    a = torch.ldexp(v, -e)
    step = 0.5 + 0.5 * (a.abs() >= 2.0) + (a.abs() >= 4.0)
    return torch.ldexp((torch.round(a / step) * step).clamp(-6.0, 6.0), e).flatten(-2)


def _plain_weight(w):
    words, scales = w
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32)
    codes = (words.unsqueeze(-1) >> shift) & 15
    v = torch.tensor(E2M1, device=words.device)[codes].flatten(-2).unflatten(-1, (-1, 32))
    return torch.ldexp(v, scales.unsqueeze(-1).int() - 127).flatten(-2)


def _plain_scores(logits, scoring):
    l = logits.double()                  # a border between two experts is decided in 64 bits
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-l))
    p = torch.exp(l - l.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_route(st):
    how, l = st["how"], st["logits"]
    s = _plain_scores(l, how["scoring"])
    key = s if st["bias"] is None else s + st["bias"].double()
    if how["groups"] > 1:
        by = key.unflatten(1, (how["groups"], -1))
        best = torch.sort(by, dim=-1, descending=True).values[..., :2].sum(-1)
        order = torch.sort(best, dim=-1, descending=True, stable=True).indices
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(
            1, order[:, :how["topk_groups"]], True)
        key = torch.where(kept.unsqueeze(2), by, -math.inf).flatten(1)
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :how["top_k"]].contiguous()
    w = s.gather(1, ids)
    if how["renormalize"]:
        w = w / (w.sum(-1, keepdim=True) + EPS)
    return (w * how["scale"]).float(), ids


def _plain_route_grad(st, ids):
    how, l = st["how"], st["logits"]
    s, dw = _plain_scores(l, how["scoring"]), st["dw"].double() * how["scale"]
    picked = s.gather(1, ids)
    if how["renormalize"]:
        total = picked.sum(-1, keepdim=True) + EPS
        dw = (dw - (dw * picked).sum(-1, keepdim=True) / total) / total
    ds = torch.zeros_like(s).scatter_(1, ids, dw)
    if how["scoring"] == "sigmoid":
        dl = ds * s * (1.0 - s)
    else:
        dl = s * (ds - (ds * s).sum(-1, keepdim=True))
    return dl.to(l.dtype)


def _plain_moe(st):
    x, ids, rows = st["x"], st["ids"], st["rows"]
    t, k = ids.shape
    gate_up, down = _plain_weight(st["gate_up"]), _plain_weight(st["down"])
    e, _, h = gate_up.shape
    flat = ids.flatten()
    expert, order = torch.sort(flat, stable=True)
    first = torch.searchsorted(expert, torch.arange(e, device=x.device))
    slot = expert * rows + torch.arange(t * k, device=x.device) - first[expert]
    xs = torch.zeros((e * rows, h), device=x.device)
    xs[slot] = _plain_rounded(x)[torch.div(order, k, rounding_mode="floor")]
    both = torch.bmm(gate_up, xs.view(e, rows, h).transpose(1, 2).contiguous())
    gate, up = both.chunk(2, 1)
    act = (gate / (1.0 + torch.exp(-gate)) * up).transpose(1, 2).contiguous()
    y = torch.bmm(down, _plain_rounded(act).transpose(1, 2).contiguous())
    y = y.transpose(1, 2).reshape(e * rows, h)
    where = torch.empty_like(slot).scatter_(0, order, slot)
    out = (y[where].view(t, k, h) * st["probs"].unsqueeze(2)).sum(1)
    return out.to(x.dtype)


def _plain(st):
    path = st["path"]
    if path == "quantize":
        return [_plain_rounded(st["x"]).to(st["x"].dtype)]
    if path == "gemm":
        return [(_plain_rounded(st["x"]) @ _plain_weight(st["w"]).t()).to(st["x"].dtype)]
    if path == "gemm_bwd":
        return [(st["dy"].float() @ _plain_weight(st["w"])).to(st["dy"].dtype)]
    if path == "moe":
        return [_plain_moe(st)]
    w, ids = _plain_route(st)
    return [w, ids] if path == "route" else [w, ids, _plain_route_grad(st, ids)]


# ------------------------------------------------------------ the framework's
def _load():
    pkg = str(Path(__file__).resolve().parent.parent / "metal-marlin_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mmfp4
    return mmfp4


def _own(st):
    mm, path = _load(), st["path"]
    if path == "quantize":
        words, scales = mm.mxfp4_quantize(st["x"])
        return [mm.mxfp4_dequantize(words, scales, st["x"].dtype)]
    if path == "gemm":
        return [mm.mxfp4_gemm(st["x"], *st["w"])]
    if path == "gemm_bwd":
        return [mm.mxfp4_gemm_backward(st["dy"], *st["w"])]
    if path == "moe":
        return [mm.moe_mlp_mxfp4(st["x"], *st["gate_up"], *st["down"], st["ids"], st["probs"])]
    how = st["how"]
    w, ids = mm.moe_route(st["logits"], how["top_k"], scoring=how["scoring"], bias=st["bias"],
                          num_groups=how["groups"], topk_groups=how["topk_groups"],
                          renormalize=how["renormalize"], scale=how["scale"])
    if path == "route":
        return [w, ids]
    return [w, ids, mm.moe_route_backward(st["dw"], st["logits"], ids, scoring=how["scoring"],
                                          renormalize=how["renormalize"], scale=how["scale"])]


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------- its floor
def _packed(rows, k):
    return rows * k // 2 + rows * k // 32


def work(case):
    path, size = case["path"], 4 if case["type"] == "fp32" else 2
    if path == "quantize":
        r, k = case["rows"], case["k"]
        # in, codes and scales written and read back, values out; compare, scale, round each
        return {"bytes": 2 * size * r * k + 2 * _packed(r, k), "flops": 3 * r * k}
    if path in ("gemm", "gemm_bwd"):
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": size * m * (n + k) + _packed(n, k), "flops": 2 * m * n * k}
    if path in ("route", "route_step"):
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        both = path == "route_step"
        return {"bytes": (3 if both else 1) * size * t * e + (28 if both else 12) * t * k,
                "flops": (20 if both else 10) * t * e}
    t, e, h, i, k = (case[v] for v in ("tokens", "experts", "hidden", "inter", "top_k"))
    used = e * (1.0 - (1.0 - 1.0 / e) ** (t * k))          # experts that some token visits
    return {"bytes": int(used * (_packed(2 * i, h) + _packed(h, i))) + 2 * size * t * h +
            12 * t * k, "flops": 6 * t * k * h * i}


# --------------------------------------------------------- the 64-bit answer
def _rounded64(x):
    """Every value to the nearest of the block's sixteen, ties to the even code."""
    shape, v = x.shape, x.double().reshape(-1, 32)
    top = v.abs().max(1, keepdim=True).values
    scale = torch.exp2(torch.floor(torch.log2(top.clamp_min(2.0 ** -125))) - 2)
    mids = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), dtype=torch.float64,
                        device=x.device)
    a = (v / scale).abs()
    code = torch.bucketize(a, mids)                        # a tie: the lower code
    up = (code < 7) & (a == mids[code.clamp_max(6)]) & (code % 2 == 1)
    grid = torch.tensor(E2M1[:8], dtype=torch.float64, device=x.device)
    return (torch.where(v < 0, -1.0, 1.0) * grid[code + up] * scale).reshape(shape)


def _weight64(w):
    words, scales = w[0].long() & 0xFFFFFFFF, w[1].double()
    k = 8 * words.shape[-1]
    out = torch.empty((*words.shape[:-1], k), dtype=torch.float64, device=words.device)
    table = torch.tensor(E2M1, dtype=torch.float64, device=words.device)
    for i in range(8):
        out[..., i::8] = table[(words >> (4 * i)) & 15]
    return out * torch.exp2(scales - 127).repeat_interleave(32, -1)


def _route64(st):
    how, l = st["how"], st["logits"].double()
    s = torch.sigmoid(l) if how["scoring"] == "sigmoid" else torch.softmax(l, -1)
    key = s if st["bias"] is None else s + st["bias"].double()
    t, e = l.shape
    n = e // how["groups"]
    if how["groups"] > 1:
        best = key.view(t, -1, n).topk(min(2, n), -1).values.sum(-1)
        lead = best.unsqueeze(1) - best.unsqueeze(2)       # [t, g, other]
        lower = torch.arange(how["groups"], device=l.device)
        ahead = (lead > 0) | ((lead == 0) & (lower.unsqueeze(0) < lower.unsqueeze(1)).t())
        out = ahead.transpose(1, 2).sum(1) >= how["topk_groups"]
        key = key.masked_fill(out.repeat_interleave(n, 1), -math.inf)
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :how["top_k"]]
    w = s.gather(1, ids)
    return s, ids, w


def exact(case, seed):
    st, path = prepare(case, seed), case["path"]
    if path == "quantize":
        return [_rounded64(st["x"])]
    if path == "gemm":
        return [_rounded64(st["x"]) @ _weight64(st["w"]).t()]
    if path == "gemm_bwd":
        return [st["dy"].double() @ _weight64(st["w"])]
    if path in ("route", "route_step"):
        how = st["how"]
        s, ids, w = _route64(st)
        c = how["scale"] / ((w.sum(-1, keepdim=True) + EPS) if how["renormalize"] else 1.0)
        if path == "route":
            return [w * c, None]
        leaf = st["logits"].double().requires_grad_(True)
        p = torch.sigmoid(leaf) if how["scoring"] == "sigmoid" else torch.softmax(leaf, -1)
        u = p.gather(1, ids)
        u = how["scale"] * (u / (u.sum(-1, keepdim=True) + EPS) if how["renormalize"] else u)
        dl, = torch.autograd.grad((u * st["dw"].double()).sum(), leaf)
        return [w * c, None, dl]
    x, ids, probs = _rounded64(st["x"]), st["ids"], st["probs"].double()
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if token.numel() == 0:
            continue
        gate, up = (x[token] @ _weight64([v[e] for v in st["gate_up"]]).t()).chunk(2, 1)
        act = _rounded64(gate * torch.sigmoid(gate) * up)
        y = act @ _weight64([v[e] for v in st["down"]]).t()
        out.index_add_(0, token, y * probs[token, slot].unsqueeze(1))
    return [out]
