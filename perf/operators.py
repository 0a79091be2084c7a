"""Cases that measure the 8-bit operators of `witchcraft_b200.fp8`: rows in
float8_e4m3fn with one f32 scale per 128 columns, weights with one per
128 x 128 block.

Operators ("op" of a case):
  norm    T5 RMSNorm with the residual addition before it and 8-bit rows out
  rows    rows of f32 / f16 / bf16 to 8 bits
  weight  a weight matrix to 8 bits (once per matrix, when a model is loaded)
  matmul  rows times weights, with or without a residual added to the result
  gated   act(rows . gate^T) * (rows . up^T), to 16 bits or to 8-bit rows

`run` computes a case in its plain form (elementary torch operations in f32),
or with `own` set through the package; `exact` is the definition in f64.
"""
import math

import torch

own = False

BLOCK = 128          # columns (and weight rows) that share a scale
E4M3_MAX = 448.0     # largest finite float8_e4m3fn
TINY = 2.0 ** -126   # smallest scale (smallest normal f32): rows of zeros
EPS = 1e-6           # T5 layer_norm_epsilon

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # queries: 32 tokens, model width 768, between the O projection and the feed-forward
        {"name": "norm_query", "op": "norm", "m": 32, "k": 768, "type": "f32", "delta": "f32"},
        # a bulk batch of 16,384 tokens at the encoder's width; the sub-layer's output comes in f16
        {"name": "norm_bulk", "op": "norm", "m": 16384, "k": 768, "type": "f32", "delta": "f16"},
        # a wider bf16 residual stream, odd row count, last block not full
        {"name": "norm_wide", "op": "norm", "m": 4095, "k": 5000, "type": "bf16", "delta": "bf16"},
        # attention output of a bulk batch on its way to the O projection
        {"name": "rows_attention", "op": "rows", "m": 16384, "k": 768, "type": "f16"},
        # the gate matrix of a feed-forward block as a model is loaded
        {"name": "weight_load", "op": "weight", "m": 2048, "k": 768, "type": "f32"},
        # Q, K and V of 32 query tokens
        {"name": "matmul_query", "op": "matmul", "m": 32, "k": 768, "n": 2304, "out": "f16", "residual": False},
        # one token against a wide matrix: the weights' bytes are the work
        {"name": "matmul_token", "op": "matmul", "m": 1, "k": 4096, "n": 12288, "out": "bf16", "residual": False},
        # a ragged batch, no size a multiple of a tile, f32 result
        {"name": "matmul_odd", "op": "matmul", "m": 1337, "k": 1000, "n": 1100, "out": "f32", "residual": False},
        # the feed-forward's second product of a bulk batch, added to the residual stream
        {"name": "matmul_residual", "op": "matmul", "m": 16384, "k": 2048, "n": 768, "out": "f32", "residual": True},
        # a large square-ish layer
        {"name": "matmul_large", "op": "matmul", "m": 8192, "k": 4096, "n": 8192, "out": "f16", "residual": False},
        # gated feed-forward of 32 query tokens, 8-bit rows for the product that follows
        {"name": "gated_query", "op": "gated", "m": 32, "k": 768, "n": 2048, "out": "fp8", "act": "gelu"},
        # the same for a bulk batch
        {"name": "gated_bulk", "op": "gated", "m": 16384, "k": 768, "n": 2048, "out": "fp8", "act": "gelu"},
    ]


def _size(rng, lo, hi):
    """Log-uniform whole number; half of them multiples of 64, as model sizes are."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["norm", "norm", "rows", "weight", "matmul", "matmul", "matmul", "matmul", "gated", "gated"])
    while True:
        m, k = _size(rng, 1, 16384), _size(rng, 64, 8192)
        if op in ("norm", "rows", "weight"):
            if m * k > 4095 * 5000:
                continue
            case = {"op": op, "m": m, "k": k, "type": rng.choice(["f32", "f16", "bf16"])}
            if op == "norm":
                case["delta"] = rng.choice(["none", case["type"], "f16" if case["type"] == "f32" else case["type"]])
            return case
        n = _size(rng, 64, 8192)
        wide = 2 if op == "gated" else 1
        if m * n * wide > 8192 * 8192 or m * n * k * wide > 8192 * 4096 * 8192:
            continue
        if op == "matmul":
            out = rng.choice(["f16", "bf16", "f32"])
            return {"op": op, "m": m, "k": k, "n": n, "out": out, "residual": rng.random() < 0.4}
        return {"op": op, "m": m, "k": k, "n": n, "out": rng.choice(["fp8", "fp8", "f16", "bf16"]),
                "act": rng.choice(["gelu", "gelu", "silu"])}


# ---------------------------------------------------------------- plain form

def _blocks(v):
    """[m, k] -> [m, blocks, 128], zeros past k."""
    m, k = v.shape
    nb = -(-k // BLOCK)
    return torch.nn.functional.pad(v, (0, nb * BLOCK - k)).view(m, nb, BLOCK)


def _plain_rows(v):
    """f32 rows -> e4m3 codes and the scale of each 128 columns."""
    b = _blocks(v)
    scales = (b.abs().amax(-1) / E4M3_MAX).clamp_min(TINY)
    codes = (b / scales[..., None]).clamp(-E4M3_MAX, E4M3_MAX).view(v.shape[0], -1)[:, :v.shape[1]]
    return codes.to(torch.float8_e4m3fn), scales


def _plain_weight(w):
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    b = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    scales = (b.abs().amax((1, 3)) / E4M3_MAX).clamp_min(TINY)
    codes = (b / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return codes.view(nb * BLOCK, kb * BLOCK)[:n, :k].to(torch.float8_e4m3fn), scales


def _plain_values(codes, scales, rows):
    """The f32 values that codes stand for; `rows`: rows that share a row of scales."""
    s = scales.repeat_interleave(rows, 0)[:codes.shape[0]].repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.float() * s


def _plain_act(g, act):
    if act == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))


def _plain(s):
    op = s["op"]
    if op == "norm":
        t = s["x"].float()
        if s["delta"] is not None:
            t = t + s["delta"].float()
        y = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * s["w"]
        codes, scales = _plain_rows(y)
        return (codes, scales) if s["delta"] is None else (t.to(s["x"].dtype), codes, scales)
    if op == "rows":
        return _plain_rows(s["x"].float())
    if op == "weight":
        return _plain_weight(s["x"].float())
    a = _plain_values(s["a"], s["sa"], 1)
    if op == "matmul":
        y = a @ _plain_values(s["w"], s["sw"], BLOCK).T
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(s["out"])
    h = _plain_act(a @ _plain_values(s["w"], s["sw"], BLOCK).T, s["act"]) * (a @ _plain_values(s["up"], s["sup"], BLOCK).T)
    return _plain_rows(h) if s["out"] is None else h.to(s["out"])


# ---------------------------------------------------------------- inputs

def _stored(codes):
    """Codes as the operators hand them on: rows start at multiples of 16 bytes."""
    m, k = codes.shape
    t = torch.zeros(m, -(-k // 16) * 16, dtype=torch.uint8, device=codes.device).view(torch.float8_e4m3fn)[:, :k]
    t.copy_(codes)
    return t


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    m, k, op = case["m"], case["k"], case["op"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def channels():
        """Per-channel spread of transformer activations: a few columns far above the rest."""
        c = 0.5 + torch.rand(k, generator=g, device="cuda")
        c[torch.randint(0, k, (max(1, k // 100),), generator=g, device="cuda")] *= 20
        return c

    if op in ("norm", "rows", "weight"):
        x = normal(m, k) * (0.02 if op == "weight" else channels())
        s = {"op": op, "x": x.to(TYPES[case["type"]])}
        if op == "norm":
            s["w"] = 1 + 0.1 * normal(k)
            s["delta"] = None if case["delta"] == "none" else normal(m, k).to(TYPES[case["delta"]])
        return s
    x = normal(m, k) * channels()
    a, sa = _plain_rows(x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))
    spread = 1 / math.sqrt(k)   # results of about unit size, as trained weights give

    def weight():
        w, sw = _plain_weight(normal(case["n"], k) * spread)
        return _stored(w), sw

    s = {"op": op, "a": _stored(a), "sa": sa, "out": TYPES.get(case["out"])}
    s["w"], s["sw"] = weight()
    if op == "gated":
        s["up"], s["sup"] = weight()
        s["act"] = case["act"]
    else:
        s["residual"] = normal(m, case["n"]).to(s["out"]) if case["residual"] else None
    return s


def run(state):
    if not own:
        return _plain(state)
    from witchcraft_b200 import fp8
    s, op = state, state["op"]
    if op == "norm":
        return fp8.rmsnorm(s["x"], s["w"], EPS, s["delta"])
    if op == "rows":
        return fp8.quantize(s["x"])
    if op == "weight":
        return fp8.quantize_weight(s["x"])
    if op == "matmul":
        return fp8.matmul(s["a"], s["sa"], s["w"], s["sw"], s["out"], s["residual"])
    return fp8.gated_matmul(s["a"], s["sa"], s["w"], s["sw"], s["up"], s["sup"], s["out"], s["act"])


# ---------------------------------------------------------------- work and definition

def work(case):
    m, k, op = case["m"], case["k"], case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    kb = -(-k // BLOCK)
    if op in ("norm", "rows", "weight"):
        scales = 4 * kb * (-(-m // BLOCK) if op == "weight" else m)
        total = m * k * size[case["type"]] + m * k + scales
        if op == "norm":
            total += 4 * k
            if case["delta"] != "none":
                total += m * k * (size[case["delta"]] + size[case["type"]])
        return {"bytes": total, "flops": (8 if op == "norm" else 3) * m * k}
    n, mats = case["n"], 2 if op == "gated" else 1
    nb = -(-n // BLOCK)
    total = m * k + 4 * m * kb + mats * (n * k + 4 * nb * kb)
    total += m * n + 4 * m * nb if case["out"] == "fp8" else m * n * size[case["out"]]
    if op == "matmul" and case["residual"]:
        total += m * n * size[case["out"]]
    return {"bytes": total, "flops": 2 * m * n * k * mats}


def _exact_codes(v, group):
    """f64 [r, c] -> (values rounded to e4m3, scales), one scale per `group` rows x 128 columns."""
    r, c = v.shape
    rb, cb = (r + group - 1) // group, (c + BLOCK - 1) // BLOCK
    ri = torch.arange(r, device=v.device) // group
    ci = torch.arange(c, device=v.device) // BLOCK
    top = torch.zeros(r, cb, dtype=torch.float64, device=v.device)
    top.scatter_reduce_(1, ci.expand(r, c), v.abs(), "amax")
    best = torch.zeros(rb, cb, dtype=torch.float64, device=v.device)
    best.scatter_reduce_(0, ri[:, None].expand(r, cb), top, "amax")
    scales = torch.clamp(best / 448, min=2.0 ** -126)
    q = v / scales[ri][:, ci]
    # round to 3 fraction bits at the value's exponent (at least 2^-6: subnormals), ties to even
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.clamp(torch.round(q / step) * step, -448, 448), scales


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "norm":
        t = s["x"].double() if s["delta"] is None else s["x"].double() + s["delta"].double()
        y = t * torch.rsqrt(t.square().sum(1, keepdim=True) / t.shape[1] + EPS) * s["w"].double()
        codes, scales = _exact_codes(y, 1)
        return (codes, scales) if s["delta"] is None else (t, codes, scales)
    if op in ("rows", "weight"):
        return _exact_codes(s["x"].double(), 1 if op == "rows" else BLOCK)

    def product(w, sw):
        """Sum over the 128-column blocks of scaled products."""
        y = torch.zeros(s["a"].shape[0], w.shape[0], dtype=torch.float64, device=w.device)
        rows = torch.arange(w.shape[0], device=w.device) // BLOCK
        for b in range(sw.shape[1]):
            cols = slice(b * BLOCK, min((b + 1) * BLOCK, w.shape[1]))
            part = s["a"][:, cols].double() * s["sa"][:, b, None].double()
            y.addmm_(part, (w[:, cols].double() * sw[rows, b, None].double()).T)
        return y

    y = product(s["w"], s["sw"])
    if op == "matmul":
        return y if s["residual"] is None else y + s["residual"].double()
    up = product(s["up"], s["sup"])
    if s["act"] == "silu":
        h = y * torch.sigmoid(y) * up
    else:
        h = y * torch.sigmoid(2 * 0.7978845608028654 * (y + 0.044715 * y ** 3)) * up
    return _exact_codes(h, 1) if s["out"] is None else h
