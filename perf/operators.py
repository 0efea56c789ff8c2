"""The operators that train and serve low-rank adapters on 4-bit weights, and what is
measured of them.  A case is a dict of plain values; its "path" says what runs:

  lora        the adapters of many requests added to a shared projection's output
  lora_bwd    the gradients of that: of the input, and of both factors of every adapter
  linear_bwd  the input gradient of one quantized linear layer (FP4 or INT4)
  qkv_bwd     the input gradient of the three projections that share an input
  gated       gate and up projections, SiLU and product, keeping what the backward needs
  gated_bwd   the input gradient of that block
  gated_step  both, one after the other, as a training step runs them

Weights are N(0, 0.02) quantized in groups along K, activations N(0, 1), gradients
N(0, 1e-3) (a loss scale is part of them), adapters as they are after some training:
the first factor N(0, 1 / sqrt(K)), the second N(0, 0.02), scaled by 1 or 2.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0,
        -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    # hidden 4096, 1024 k/v columns, intermediate 14336: the benchmark's dense model
    return [
        # one token of one request, where launch latency counts
        {"name": "lora_t1", "path": "lora", "type": "fp16", "tokens": 1, "requests": 1, "bare": 0,
         "adapters": 8, "rank": 16, "k": 4096, "n": 4096},
        # a decode batch: every request with an adapter of its own
        {"name": "lora_t32", "path": "lora", "type": "bf16", "tokens": 32, "requests": 32,
         "bare": 0, "adapters": 64, "rank": 16, "k": 4096, "n": 6144},
        # prompts of seven requests in one batch, two of them without an adapter
        {"name": "lora_t1111", "path": "lora", "type": "fp16", "tokens": 1111, "requests": 7,
         "bare": 2, "adapters": 4, "rank": 64, "k": 14336, "n": 4096},
        # adapters of several users trained together, an odd number of tokens, a small rank
        {"name": "lora_bwd_t777", "path": "lora_bwd", "type": "bf16", "tokens": 777,
         "requests": 5, "bare": 0, "adapters": 3, "rank": 8, "k": 2048, "n": 5632},
        # fine-tuning one adapter on a long batch
        {"name": "lora_bwd_t4096", "path": "lora_bwd", "type": "fp16", "tokens": 4096,
         "requests": 1, "bare": 0, "adapters": 1, "rank": 16, "k": 4096, "n": 14336},
        # the gradient of one token's input (a soft prompt, an attribution)
        {"name": "linear_bwd_m1", "path": "linear_bwd", "type": "fp16", "fmt": "fp4", "m": 1,
         "n": 4096, "k": 4096, "group": 128},
        # a short batch through asymmetric INT4 weights
        {"name": "linear_bwd_int4_m300", "path": "linear_bwd", "type": "bf16", "fmt": "int4",
         "m": 300, "n": 4096, "k": 4096, "group": 128},
        # a full training batch through the widest layer
        {"name": "linear_bwd_m2048", "path": "linear_bwd", "type": "fp16", "fmt": "fp4",
         "m": 2048, "n": 14336, "k": 4096, "group": 128},
        # the attention projections of a batch with an odd number of tokens
        {"name": "qkv_bwd_m509", "path": "qkv_bwd", "type": "bf16", "m": 509, "hidden": 4096,
         "kv": 1024, "group": 128},
        # forward of a short batch
        {"name": "gated_m100", "path": "gated", "type": "fp16", "m": 100, "n": 14336, "k": 4096,
         "group": 128},
        # backward on a smaller model with smaller groups
        {"name": "gated_bwd_m1000", "path": "gated_bwd", "type": "bf16", "m": 1000, "n": 5632,
         "k": 2048, "group": 64},
        # the largest: the block's whole training step on a full batch
        {"name": "gated_step_m2048", "path": "gated_step", "type": "fp16", "m": 2048, "n": 14336,
         "k": 4096, "group": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(("lora", "lora", "lora", "lora_bwd", "lora_bwd", "linear_bwd", "linear_bwd",
                       "qkv_bwd", "gated", "gated_bwd", "gated_step"))
    case = {"path": path, "type": rng.choice(("fp16", "bf16"))}
    if path in ("lora", "lora_bwd"):
        tokens = _log(rng, 1, 8192)
        requests = tokens if tokens <= 256 and rng.random() < 0.7 else \
            min(tokens, _log(rng, 1, 32))
        rank = rng.choice((4, 8, 16, 16, 32, 64, 128, rng.randint(1, 64)))
        k, n = 8 * _log(rng, 64, 1792), 8 * _log(rng, 64, 1792) + rng.choice((0, 0, 0, 4, 1))
        # the plain form multiplies with every adapter: at most the largest's work
        adapters = min(_log(rng, 1, 64), max(1, 150_000_000_000 // (tokens * rank * (k + n))))
        return {**case, "tokens": tokens, "requests": requests,
                "bare": rng.choice((0, 0, requests // 4)), "adapters": adapters, "rank": rank,
                "k": k, "n": n}
    case["group"] = rng.choice((32, 64, 128, 128, 128))
    if path == "qkv_bwd":
        hidden = 128 * rng.randint(8, 32)
        return {**case, "m": _log(rng, 1, 4096), "hidden": hidden,
                "kv": rng.choice((256, 512, 1024, hidden))}
    k = 128 * _log(rng, 4, 64)
    n = 8 * _log(rng, 64, 1792)
    if path == "linear_bwd":
        n += rng.choice((0, 0, 0, 4, 1))
        case["fmt"] = rng.choice(("fp4", "fp4", "int4"))
    m = min(_log(rng, 1, 8192), 120_000_000_000 // (n * k))   # at most the largest's work
    return {**case, "m": m, "n": n, "k": k}


# ------------------------------------------------------------------- inputs
class _Inputs:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.gen = torch.Generator(self.dev).manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float16):
        return (torch.randn(shape, generator=self.gen, device=self.dev) * std).to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device=self.dev)

    def fp4(self, k, n, group):
        """A quantized matrix: words [K/8, N], scales [K/g, N]."""
        w = torch.randn((k // group, group, n), generator=self.gen, device=self.dev) * 0.02
        amax = w.abs().amax(1).clamp_min(1e-7)
        v = w / amax.unsqueeze(1) * 6.0
        mids = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device=self.dev)
        codes = torch.bucketize(v.abs(), mids, out_int32=True) + 8 * (v < 0)
        return _pack(codes.reshape(k, n)), (amax / 6.0).half()

    def int4(self, k, n, group):
        """Words, scales and zero points of an asymmetric matrix."""
        w = torch.randn((k // group, group, n), generator=self.gen, device=self.dev) * 0.02
        lo, hi = w.amin(1), w.amax(1)
        s = ((hi - lo) / 15.0).clamp_min(1e-7).half()
        z = torch.round(-lo / s.float()).clamp(0, 15)
        q = torch.round(w / s.float().unsqueeze(1) + z.unsqueeze(1)).clamp(0, 15)
        return _pack(q.reshape(k, n)), s, z.half()


def _pack(codes):
    c = codes.to(torch.int32).unflatten(0, (-1, 8))
    shift = 4 * torch.arange(8, device=c.device, dtype=torch.int32).view(8, 1)
    return torch.sum(c << shift, dim=1, dtype=torch.int32).contiguous()


def _ids(case, make):
    """Adapter of every token: the requests' tokens lie one after another, in lengths that
    differ; the first `bare` requests have none (-1), the others go round the adapters."""
    t, r = case["tokens"], case["requests"]
    cuts = torch.sort(make.order(t - 1)[:r - 1] + 1).values if r > 1 else \
        torch.zeros(0, dtype=torch.int64, device=make.dev)
    request = torch.bucketize(torch.arange(t, device=make.dev), cuts, right=True)
    which = make.order(case["adapters"])[(request - case["bare"]) % case["adapters"]]
    return torch.where(request < case["bare"], -1, which).to(torch.int32)


def prepare(case, seed):
    make, dt = _Inputs(seed), TYPES[case["type"]]
    path = case["path"]
    if path in ("lora", "lora_bwd"):
        t, k, n, r, l = (case[v] for v in ("tokens", "k", "n", "rank", "adapters"))
        st = {"x": make.normal(t, k, dtype=dt),
              "a": make.normal(l, r, k, std=k ** -0.5, dtype=dt),
              "b": make.normal(l, n, r, std=0.02, dtype=dt),
              "ids": _ids(case, make),
              "scaling": 1.0 + (make.order(l) % 2).float()}
        if path == "lora":
            return {**st, "path": path, "base": make.normal(t, n, dtype=dt)}
        return {**st, "path": path, "dy": make.normal(t, n, std=1e-3, dtype=dt),
                "dx_base": make.normal(t, k, std=1e-3, dtype=dt)}
    g, m = case["group"], case["m"]
    if path == "qkv_bwd":
        ns = (case["hidden"], case["kv"], case["kv"])
        return {"path": path, "group": g,
                "w": [make.fp4(case["hidden"], n, g) for n in ns],
                "dy": [make.normal(m, n, std=1e-3, dtype=dt) for n in ns]}
    k, n = case["k"], case["n"]
    if path == "linear_bwd":
        return {"path": path, "group": g, "w": getattr(make, case["fmt"])(k, n, g),
                "dy": make.normal(m, n, std=1e-3, dtype=dt)}
    st = {"path": path, "group": g, "gate": make.fp4(k, n, g), "up": make.fp4(k, n, g)}
    if path != "gated_bwd":
        st["x"] = make.normal(m, k, dtype=dt)
    if path == "gated_bwd":
        st["gate_up"] = make.normal(m, 2 * n)
    if path != "gated":
        st["dh"] = make.normal(m, n, std=1e-3, dtype=dt)
    return st


# ---------------------------------------------------------------- plain form
def _dequant(w, group):
    """The fp16 weights [K, N] that the packed words stand for, as fp32."""
    words, scales = w[0], w[1]
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32).view(8, 1)
    codes = ((words.unsqueeze(1) >> shift) & 15).flatten(0, 1)
    s = scales.float().repeat_interleave(group, 0)
    if len(w) == 3:
        return ((codes - w[2].float().repeat_interleave(group, 0)) * s).half().float()
    return (torch.tensor(E2M1, device=words.device)[codes] * s).half().float()


def _plain_hidden(v, w, st):
    """s v W_a^T of every token under every adapter, zero but for its own: [T, L * r]."""
    l, r = w.shape[:2]
    mine = (st["ids"].unsqueeze(1) == torch.arange(l, device=v.device)).float()
    h = (v @ w.float().reshape(l * r, -1).t()).unflatten(1, (l, r))
    return (h * (mine * st["scaling"]).unsqueeze(2)).flatten(1)


def _plain_gated(st, dt):
    x, g = st["x"].half().float(), st["group"]
    gate, up = x @ _dequant(st["gate"], g), x @ _dequant(st["up"], g)
    h = gate / (1.0 + torch.exp(-gate)) * up
    return [h.half(), torch.cat([gate, up], 1).half()]


def _plain_gated_bwd(st, gate_up):
    gate, up = gate_up.float().chunk(2, 1)
    dh, sig = st["dh"].float(), 1.0 / (1.0 + torch.exp(-gate))
    dgate = dh * up * sig * (1.0 + gate * (1.0 - sig))
    dup = dh * gate * sig
    dx = dgate @ _dequant(st["gate"], st["group"]).t() + dup @ _dequant(st["up"], st["group"]).t()
    return dx.to(st["dh"].dtype)


def _plain(st):
    path = st["path"]
    if path == "lora":
        h = _plain_hidden(st["x"].float(), st["a"], st)
        out = st["base"].float() + h @ st["b"].float().transpose(1, 2).flatten(0, 1)
        return [out.to(st["x"].dtype)]
    if path == "lora_bwd":
        x, dy, a = st["x"].float(), st["dy"].float(), st["a"].float()
        bt = st["b"].transpose(1, 2)                       # [L, r, N]
        h, dh = _plain_hidden(x, a, st), _plain_hidden(dy, bt, st)
        dx = st["dx_base"].float() + dh @ a.flatten(0, 1)
        da = (dh.t() @ x).view_as(a)
        db = (h.t() @ dy).view(bt.shape).transpose(1, 2)
        dt = st["x"].dtype
        return [dx.to(dt), da.to(dt), db.to(dt).contiguous()]
    if path == "linear_bwd":
        dx = st["dy"].float() @ _dequant(st["w"], st["group"]).t()
        return [dx.to(st["dy"].dtype)]
    if path == "qkv_bwd":
        (wq, wk, wv), (dq, dk, dv), g = st["w"], st["dy"], st["group"]
        dx = dq.float() @ _dequant(wq, g).t() + dk.float() @ _dequant(wk, g).t() + \
            dv.float() @ _dequant(wv, g).t()
        return [dx.to(dq.dtype)]
    if path == "gated":
        return _plain_gated(st, st["x"].dtype)
    if path == "gated_bwd":
        return [_plain_gated_bwd(st, st["gate_up"])]
    h, gate_up = _plain_gated(st, st["x"].dtype)
    return [h, gate_up, _plain_gated_bwd(st, gate_up)]


# ------------------------------------------------------------ the framework's
def _mmfp4():
    pkg = str(Path(__file__).resolve().parent.parent / "metal-marlin_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mmfp4
    return mmfp4


def _own(st):
    mm, path = _mmfp4(), st["path"]
    if path == "lora":
        return [mm.lora_add(st["base"], st["x"], st["a"], st["b"], st["ids"], st["scaling"])]
    if path == "lora_bwd":
        return list(mm.lora_backward(st["dy"], st["x"], st["a"], st["b"], st["ids"],
                                     st["scaling"], dx_base=st["dx_base"]))
    g = st["group"]
    if path == "linear_bwd":
        w = st["w"]
        if len(w) == 3:
            return [mm.marlin_gemm_int4_backward(st["dy"], w[0], w[1], w[2], g)]
        return [mm.marlin_gemm_fp4_backward(st["dy"], w[0], w[1], g)]
    if path == "qkv_bwd":
        (wq, wk, wv), (dq, dk, dv) = st["w"], st["dy"]
        return [mm.mmfp4_fused_qkv_backward(dq, dk, dv, *wq, *wk, *wv, g)]
    h, gate_up, out = None, st.get("gate_up"), []
    if path != "gated_bwd":
        h, gate_up = mm.fused_gate_up_swiglu(st["x"], *st["gate"], *st["up"], g)
        out = [h, gate_up]
    if path != "gated":
        out.append(mm.fused_gate_up_swiglu_backward(st["dh"], gate_up, *st["gate"], *st["up"], g))
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------- its floor
def _words(k, n, group, int4=False):
    return k * n // 2 + (4 if int4 else 2) * (k // group) * n


def work(case):
    path = case["path"]
    if path in ("lora", "lora_bwd"):
        t, k, n, r, l = (case[v] for v in ("tokens", "k", "n", "rank", "adapters"))
        used = min(l, case["requests"] - case["bare"])
        factors = 2 * used * r * (k + n)
        if path == "lora":
            return {"bytes": 2 * t * (k + 2 * n) + factors + 4 * t, "flops": 2 * t * r * (k + n)}
        return {"bytes": 2 * t * (3 * k + n) + factors + 2 * l * r * (k + n) + 4 * t,
                "flops": 2 * t * r * (3 * k + 2 * n)}
    m, g = case["m"], case["group"]
    if path == "qkv_bwd":
        k, n = case["hidden"], case["hidden"] + 2 * case["kv"]
        return {"bytes": 2 * m * (k + n) + _words(k, n, g), "flops": 2 * m * n * k}
    k, n = case["k"], case["n"]
    if path == "linear_bwd":
        return {"bytes": 2 * m * (k + n) + _words(k, n, g, case["fmt"] == "int4"),
                "flops": 2 * m * n * k}
    half = {"bytes": 2 * m * (k + 3 * n) + 2 * _words(k, n, g), "flops": 4 * m * n * k}
    return {v: half[v] * (2 if path == "gated_step" else 1) for v in half}


# --------------------------------------------------------- the 64-bit answer
def _weights64(w, group):
    """[K, N] in 64 bits: every weight is the fp16 nearest to (code - zero) * scale, or to
    the code's E2M1 value * scale."""
    words, scales = w[0].long() & 0xFFFFFFFF, w[1].double()
    k, n = 8 * words.shape[0], words.shape[1]
    out = torch.empty((k, n), dtype=torch.float64, device=words.device)
    table = torch.tensor(E2M1, dtype=torch.float64, device=words.device)
    rows = torch.arange(0, k, 8, device=words.device)
    for i in range(8):
        code, group_of = (words >> (4 * i)) & 15, (rows + i) // group
        v = code.double() - w[2].double()[group_of] if len(w) == 3 else table[code]
        out[i::8] = (v * scales[group_of]).half().double()
    return out


def _gated64(gate, up, dh=None):
    sig = torch.sigmoid(gate)
    if dh is None:
        return gate * sig * up
    return dh * up * (sig + gate * sig * (1 - sig)), dh * gate * sig


def exact(case, seed):
    st, path = prepare(case, seed), case["path"]
    if path in ("lora", "lora_bwd"):
        x, out = st["x"].double(), st["base" if path == "lora" else "dx_base"].double()
        da, db = torch.zeros_like(st["a"], dtype=torch.float64), \
            torch.zeros_like(st["b"], dtype=torch.float64)
        for i in range(case["adapters"]):
            rows = torch.nonzero(st["ids"] == i).flatten()
            a, b, s = st["a"][i].double(), st["b"][i].double(), st["scaling"][i].double()
            if path == "lora":
                out[rows] += s * (x[rows] @ a.t() @ b.t())
                continue
            dy = st["dy"][rows].double()
            dh = s * (dy @ b)
            out[rows] += dh @ a
            da[i], db[i] = dh.t() @ x[rows], s * (dy.t() @ (x[rows] @ a.t()))
        return [out] if path == "lora" else [out, da, db]
    g = st["group"]
    if path == "linear_bwd":
        return [st["dy"].double() @ _weights64(st["w"], g).t()]
    if path == "qkv_bwd":
        return [sum(d.double() @ _weights64(w, g).t() for d, w in zip(st["dy"], st["w"]))]
    wg, wu = _weights64(st["gate"], g), _weights64(st["up"], g)
    if path == "gated_bwd":
        gate, up = st["gate_up"].double().chunk(2, 1)
        dgate, dup = _gated64(gate, up, st["dh"].double())
        return [dgate @ wg.t() + dup @ wu.t()]
    x = st["x"].half().double()
    gate, up = x @ wg, x @ wu
    out = [_gated64(gate, up), torch.cat([gate, up], 1)]
    if path == "gated_step":
        kept = out[1].half().double().chunk(2, 1)     # the backward starts from what is kept
        dgate, dup = _gated64(*kept, st["dh"].double())
        out.append(dgate @ wg.t() + dup @ wu.t())
    return out
