"""Measured cases of the MXFP4 operators and of the MoE layer for a few tokens.

Four operators, each with a plain form in elementary torch operations and the framework's own call:

  roundtrip  quantisation of bf16 activations to MXFP4 (blocks of 32 along the last axis, e2m1 values, one power-of-two
             scale per block) and back: what a loader does with a weight and a linear layer with its input
  silu       SiLU(gate) * up, rounded to bf16 after each of the two steps, then quantised to MXFP4 and read back
  linear     y = Q(x) W^T (+ bias): x quantised to MXFP4 on the way, W held in MXFP4, fp32 sums, bf16 result
  moe        the whole mixture-of-experts layer behind the router's logits for 1 to 16 tokens: top-k routing, the chosen
             experts' SwiGLU MLPs, the weighted sum.  Experts in FP8 with 128x128 block scales or in MXFP4
"""
from __future__ import annotations

import math

import torch

own = False

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


# ---- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step's input of a linear layer of hidden size 7168: latency only
        {"name": "roundtrip_decode", "op": "roundtrip", "m": 1, "k": 7168},
        # a prefill batch of the same layer
        {"name": "roundtrip_prefill", "op": "roundtrip", "m": 8192, "k": 7168},
        # a small, odd batch between the two projections of a shared expert
        {"name": "silu_small", "op": "silu", "m": 129, "n": 2048},
        # the activation benchmark's shape: 16384 rows of 2 x 2048, a few outliers
        {"name": "silu_prefill", "op": "silu", "m": 16384, "n": 2048},
        # one token through a projection 7168 -> 4096: the weights are all there is to read
        {"name": "linear_token", "op": "linear", "m": 1, "n": 4096, "k": 7168, "bias": False},
        # a decode batch, ragged sizes, with a bias
        {"name": "linear_ragged", "op": "linear", "m": 77, "n": 2056, "k": 1440, "bias": True},
        # the dense benchmark's shape: a few hundred rows
        {"name": "linear_rows", "op": "linear", "m": 512, "n": 4096, "k": 7168, "bias": False},
        # prefill: bound by the tensor cores
        {"name": "linear_prefill", "op": "linear", "m": 8192, "n": 7168, "k": 7168, "bias": False},
        # one token, many small experts, softmax routing: latency
        {"name": "moe_token_small", "op": "moe", "t": 1, "h": 2048, "i": 768, "e": 128, "top": 8, "fmt": "fp8", "score": "softmax", "groups": 1, "keep": 1},
        # one token of the DeepSeek-V3-shaped layer, grouped sigmoid routing with a selection bias
        {"name": "moe_token_large", "op": "moe", "t": 1, "h": 7168, "i": 2048, "e": 256, "top": 8, "fmt": "fp8", "score": "sigmoid", "groups": 8, "keep": 4},
        # a handful of tokens of the Mixtral-8x7B-shaped layer with MXFP4 experts
        {"name": "moe_mixtral_mxfp4", "op": "moe", "t": 5, "h": 4096, "i": 14336, "e": 8, "top": 2, "fmt": "mxfp4", "score": "softmax", "groups": 1, "keep": 1},
        # the largest batch of the few-token form: 16 tokens over 256 experts
        {"name": "moe_batch_large", "op": "moe", "t": 16, "h": 7168, "i": 2048, "e": 256, "top": 8, "fmt": "fp8", "score": "sigmoid", "groups": 8, "keep": 4},
    ]


def _log(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["roundtrip", "silu", "linear", "linear", "moe", "moe"])
    if op == "roundtrip":
        return {"op": op, "m": _log(rng, 1, 8192), "k": _log(rng, 32, 7168, 32)}
    if op == "silu":
        return {"op": op, "m": _log(rng, 1, 16384), "n": _log(rng, 32, 2048, 32)}
    if op == "linear":
        return {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 7168, 8), "k": _log(rng, 64, 7168, 32), "bias": rng.random() < 0.5}
    score = rng.choice(["softmax", "sigmoid"])
    groups = rng.choice([1, 4, 8]) if score == "sigmoid" else 1
    return {"op": op, "t": _log(rng, 1, 16), "h": _log(rng, 512, 7168, 128), "i": _log(rng, 256, 2048, 128), "e": groups * _log(rng, 8, 256 // groups),
            "top": rng.randint(1, 8), "fmt": rng.choice(["fp8", "mxfp4"]), "score": score, "groups": groups, "keep": max(1, groups // 2)}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _mxfp4_weight(shape, gen):
    """Random MXFP4 weight [..., n, k]: packed codes uint8 [..., n, k/2] and scale bytes uint8 [..., n, k/32]; what a Gaussian
    weight of standard deviation about 0.02 looks like after quantisation."""
    *lead, k = shape
    codes = torch.empty(*lead, k // 2, dtype=torch.uint8, device="cuda")
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")

    def some(rows):
        v = torch.randn(rows, k, generator=gen, device="cuda").mul_(2.2)
        c = torch.bucketize(v.abs(), edges, out_int32=True).to(torch.uint8) | (v < 0).to(torch.uint8) << 3
        return c[:, 0::2] | c[:, 1::2] << 4

    flat = codes.view(-1, k // 2)
    step = max(1, (1 << 26) // k)
    for r in range(0, flat.shape[0], step):
        flat[r:r + step] = some(min(step, flat.shape[0] - r))
    scales = torch.randint(119, 122, (*lead, k // 32), generator=gen, device="cuda", dtype=torch.uint8)
    return codes, scales


def _fp8_weight(e, n, k, gen):
    """FP8 expert weights [e, n, k] with fp32 128x128 block scales (not powers of two, as in a checkpoint)."""
    q = torch.empty(e, n, k, dtype=torch.float8_e4m3fn, device="cuda")
    for x in range(e):
        q[x] = torch.randn(n, k, generator=gen, device="cuda").mul_(100.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    s = torch.empty(e, -(-n // 128), -(-k // 128), device="cuda").uniform_(1.5e-4, 2.5e-4, generator=gen)
    return q, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 17)
    st = dict(case)

    def acts(m, k):
        x = torch.randn(m, k, generator=gen, device="cuda")
        x = torch.where(torch.rand(m, k, generator=gen, device="cuda") < 1e-3, x * 50.0, x)      # a few outliers, as activations have
        return x.to(torch.bfloat16)

    if case["op"] in ("roundtrip", "silu"):
        m, k = (case["m"], case["k"]) if case["op"] == "roundtrip" else (case["m"], case["n"])
        st["x"] = acts(m, k if case["op"] == "roundtrip" else 2 * k)
        st["q"] = torch.empty(m, k // 2, dtype=torch.uint8, device="cuda")
        st["s"] = torch.empty(m, k // 32, dtype=torch.uint8, device="cuda")
        st["out"] = torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    elif case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        st["x"] = acts(m, k)
        st["w"], st["ws"] = _mxfp4_weight((n, k), gen)
        st["b"] = torch.randn(n, generator=gen, device="cuda").to(torch.bfloat16) if case["bias"] else None
        if own:
            from kb_nano_b200 import ops

            st["wp"] = ops.pack_mxfp4_scales(st["ws"], k)           # laid out once, when the weight is loaded
            st["q"] = torch.empty(m, k // 2, dtype=torch.uint8, device="cuda")
            st["sf"] = torch.empty(ops.packed_mxfp4_bytes(m, k), dtype=torch.uint8, device="cuda")
            st["out"] = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    else:
        t, h, i, e = case["t"], case["h"], case["i"], case["e"]
        st["x"] = torch.randn(t, h, generator=gen, device="cuda").to(torch.bfloat16)
        st["logits"] = torch.randn(t, e, generator=gen, device="cuda")
        st["bias"] = torch.randn(e, generator=gen, device="cuda").mul_(0.05) if case["score"] == "sigmoid" else None
        if case["fmt"] == "fp8":
            st["w13"], st["s13"] = _fp8_weight(e, 2 * i, h, gen)
            st["w2"], st["s2"] = _fp8_weight(e, h, i, gen)
        else:
            st["w13"], st["s13"] = _mxfp4_weight((e, 2 * i, h), gen)
            st["w2"], st["s2"] = _mxfp4_weight((e, h, i), gen)
        st["out"] = torch.empty(t, h, dtype=torch.bfloat16, device="cuda")
    return st


# ---- the operators ----------------------------------------------------------------------------------------------------

def _pow2(e):
    """Exactly 2^e in fp32 for whole e in [-127, 127], put together from its exponent bits (in two factors: 2^-127 is subnormal)."""
    half = e >> 1
    return ((half + 127) << 23).view(torch.float32) * ((e - half + 127) << 23).view(torch.float32)


def _plain_quant(y):
    """fp32 y [m, k] -> the fp32 values that its MXFP4 form stands for."""
    m, k = y.shape
    b = y.view(m, k // 32, 32)
    frac, exp = torch.frexp(b.abs().amax(dim=2, keepdim=True))      # amax = frac * 2^exp, frac in [0.5, 1)
    e = (exp - 3 + (frac > 0.75).to(torch.int32)).clamp(-127, 127)  # smallest e with amax <= 6 * 2^e
    v = b * _pow2(-e)
    a = v.abs()
    q = ((a > 0.25).float() + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) * 0.5 + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5.0)
    return (q * _pow2(e) * torch.sign(v)).view(m, k)


def _plain_unpack(codes, scales):
    """packed codes [..., k/2] and scale bytes [..., k/32] -> fp32 values [..., k]."""
    lut = torch.tensor(_E2M1, device=codes.device)
    v = torch.stack((lut[(codes & 15).int()], lut[(codes >> 4).int()]), dim=-1).flatten(-2)
    return (v.view(*scales.shape, 32) * _pow2(scales.int() - 127).unsqueeze(-1)).view(v.shape)


def _plain_fp8(q, s):
    """FP8 weights [p, n, k] and block scales [p, n/128, k/128] -> fp32 values."""
    p, n, k = q.shape
    return (q.float().view(p, n // 128, 128, k // 128, 128) * s[:, :, None, :, None]).view(p, n, k)


def _plain_route(logits, bias, case):
    """Weights [t, top] and experts [t, top]; ties go to the lowest index."""
    t, e = logits.shape
    score = torch.softmax(logits, dim=1) if case["score"] == "softmax" else torch.sigmoid(logits)
    choice = score if bias is None else score + bias
    g = case["groups"]
    if g > 1:
        per = choice.view(t, g, e // g)
        best = per.topk(min(2, e // g), dim=2).values.sum(dim=2) if bias is not None else per.amax(dim=2)
        kept = torch.zeros_like(best).scatter_(1, best.sort(dim=1, descending=True, stable=True).indices[:, : case["keep"]], 1.0)
        choice = per.masked_fill(kept.unsqueeze(2) == 0, float("-inf")).view(t, e)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, : case["top"]]
    w = score.gather(1, ids)
    return w / w.sum(dim=1, keepdim=True), ids


def run(st):
    op = st["op"]
    if own:
        from kb_nano_b200 import moe, ops

        if op == "roundtrip":
            ops.quant_mxfp4(st["x"], st["q"], st["s"])
            ops.dequant_mxfp4(st["q"], st["s"], st["out"])
        elif op == "silu":
            ops.silu_mul_quant_mxfp4(st["x"], st["q"], st["s"])
            ops.dequant_mxfp4(st["q"], st["s"], st["out"])
        elif op == "linear":
            ops.mxfp4_linear(st["x"], st["q"], st["sf"], st["w"], st["wp"], st["out"], st["b"])
        else:
            moe.few_tokens_moe(st["x"], st["logits"], st["w13"], st["s13"], st["w2"], st["s2"], st["top"], scoring=st["score"], bias=st["bias"],
                               n_group=st["groups"], topk_group=st["keep"], out=st["out"])
        return st["out"]
    if op == "roundtrip":
        return _plain_quant(st["x"].float()).to(torch.bfloat16)
    if op == "silu":
        gate, up = st["x"].float().chunk(2, dim=1)
        # the sigmoid in 64 bits: its bf16 rounding decides between neighbouring 4-bit values
        s = (gate.double() / (1.0 + torch.exp(-gate.double()))).float().to(torch.bfloat16).float()
        return _plain_quant((s * up).to(torch.bfloat16).float()).to(torch.bfloat16)
    if op == "linear":
        y = _plain_quant(st["x"].float()) @ _plain_unpack(st["w"], st["ws"]).t()
        return (y if st["b"] is None else y + st["b"].float()).to(torch.bfloat16)
    w, ids = _plain_route(st["logits"], st["bias"], st)
    t, h = st["x"].shape
    flat = ids.reshape(-1)
    x = st["x"].float().repeat_interleave(st["top"], dim=0).unsqueeze(2)                            # [t * top, h, 1]
    deq = _plain_fp8 if st["fmt"] == "fp8" else _plain_unpack
    gate, up = torch.bmm(deq(st["w13"][flat], st["s13"][flat]), x).chunk(2, dim=1)
    rows = torch.bmm(deq(st["w2"][flat], st["s2"][flat]), gate / (1.0 + torch.exp(-gate)) * up)     # [t * top, h, 1]
    return (rows.view(t, st["top"], h) * w.unsqueeze(2)).sum(dim=1).to(torch.bfloat16)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    if case["op"] in ("roundtrip", "silu"):
        n = case["m"] * (case["k"] if case["op"] == "roundtrip" else case["n"])
        inputs = 2 * n if case["op"] == "roundtrip" else 4 * n
        # input, packed form written and read again, values
        return {"bytes": inputs + 2 * n * 17 / 32 + 2 * n, "flops": 4 * n}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k * 17 / 32 + 2 * m * n, "flops": 2 * m * n * k}
    t, h, i, e, top = case["t"], case["h"], case["i"], case["e"], case["top"]
    per = 3 * h * i * (1.0 if case["fmt"] == "fp8" else 17 / 32)
    distinct = e * (1.0 - (1.0 - top / e) ** t)              # experts that t tokens choose between them, expected
    return {"bytes": distinct * per + 4 * t * h + 4 * t * e, "flops": 6 * t * top * h * i}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def _exact_pow2(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_bf16(v):
    frac, exp = torch.frexp(v)
    return torch.round(frac * 256.0) / 256.0 * _exact_pow2(exp.clamp(-1000, 1000))      # 8 significant bits, half to even


def _exact_quant(y):
    v = y.reshape(y.shape[0], -1, 32)
    top = v.abs().max(dim=2, keepdim=True).values
    e = torch.floor(torch.log2(top.clamp_min(2.0**-200))) - 2.0
    e = (e + (top > 6.0 * _exact_pow2(e))).clamp(-127, 127)             # smallest e with top <= 6 * 2^e
    scale = _exact_pow2(e)
    z = v / scale
    step = torch.where(z.abs() < 2, 0.5, torch.where(z.abs() < 4, 1.0, 2.0)).to(z.dtype)
    return (torch.round(z / step) * step * scale).reshape(y.shape)      # torch.round is half to even, as the format rounds


def _exact_values(codes, scales):
    c = torch.stack([codes % 16, codes // 16], dim=-1).reshape(*codes.shape[:-1], -1).to(torch.int64)
    sign, mag = 1.0 - 2.0 * (c // 8).double(), c % 8
    val = torch.where(mag < 2, mag.double() * 0.5, (1.0 + (mag % 2).double() * 0.5) * _exact_pow2(mag // 2 - 1))
    return sign * val * _exact_pow2(scales.to(torch.int64) - 127).repeat_interleave(32, dim=-1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "roundtrip":
        return _exact_quant(st["x"].double())
    if case["op"] == "silu":
        n = case["n"]
        gate = st["x"][:, :n].double()
        return _exact_quant(_exact_bf16(_exact_bf16(gate / (1.0 + torch.exp(-gate))) * st["x"][:, n:].double()))
    if case["op"] == "linear":
        y = torch.matmul(_exact_quant(st["x"].double()), _exact_values(st["w"], st["ws"]).t())
        return y if st["b"] is None else y + st["b"].double()
    lg, t, e = st["logits"].double(), case["t"], case["e"]
    score = torch.exp(lg - lg.logsumexp(dim=1, keepdim=True)) if case["score"] == "softmax" else 1.0 / (1.0 + torch.exp(-lg))
    pick = score + (st["bias"].double() if st["bias"] is not None else 0.0)
    if case["groups"] > 1:
        size = e // case["groups"]
        for row in range(t):
            rank = [float(pick[row, g * size:(g + 1) * size].sort(descending=True).values[:2 if st["bias"] is not None else 1].sum()) for g in range(case["groups"])]
            for g in sorted(range(case["groups"]), key=lambda j: (-rank[j], j))[case["keep"]:]:
                pick[row, g * size:(g + 1) * size] = -math.inf
    out = torch.zeros(t, case["h"], dtype=torch.float64, device="cuda")
    chosen = torch.argsort(pick, dim=1, descending=True, stable=True)[:, : case["top"]]
    for x in chosen.unique().tolist():
        rows = (chosen == x).any(dim=1).nonzero().flatten()
        if case["fmt"] == "fp8":
            a, b = (q[x].double() * s[x].double().repeat_interleave(128, dim=0).repeat_interleave(128, dim=1) for q, s in ((st["w13"], st["s13"]), (st["w2"], st["s2"])))
        else:
            a, b = (_exact_values(q[x], s[x]) for q, s in ((st["w13"], st["s13"]), (st["w2"], st["s2"])))
        both = st["x"][rows].double() @ a.t()
        g, u = both[:, : case["i"]], both[:, case["i"]:]
        wsum = score.gather(1, chosen).sum(dim=1)
        out[rows] += (score[rows, x] / wsum[rows]).unsqueeze(1) * ((g / (1.0 + torch.exp(-g)) * u) @ b.t())
    return out
