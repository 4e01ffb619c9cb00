"""MXFP4 and the MoE layer for a few tokens, restated in 64 bits for the tests (any device)."""
from __future__ import annotations

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], dtype=torch.float64)


def pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e as fp64, from the exponent bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def quant(x: torch.Tensor):
    """[M,K] -> (codes uint8 [M,K/2], scale bytes uint8 [M,K/32]): smallest 2^e >= amax / 6, nearest code, ties to even codes."""
    m, k = x.shape
    v = x.double().reshape(m, k // 32, 32)
    bad = ~torch.isfinite(v).all(dim=2)
    amax = torch.where(torch.isfinite(v), v.abs(), 0.0).amax(dim=2)
    _, ex = torch.frexp(amax)
    e = (ex - 2).double()                                        # amax < 2^ex, so 2^(ex-2) always clips nothing
    for cand in (-3, -4):
        c = (ex + cand).double()
        e = torch.where(amax <= 6.0 * pow2(c), c, e)
    e = torch.where(amax == 0, -127.0, e.clamp_min(-127.0))      # the format's smallest scale
    z = v * pow2(-e).unsqueeze(2)
    levels = E2M1[:8].to(x.device)
    d = (torch.where(torch.isfinite(z), z, 0.0).abs().unsqueeze(3) - levels).abs()
    best = d.amin(dim=3, keepdim=True)
    tie = d == best                                              # one level, or two neighbours at a midpoint
    idx = torch.arange(8, device=x.device)
    code = torch.where(tie, idx, 99).amin(dim=3)
    code = torch.where((tie.sum(dim=3) == 2) & (code % 2 == 1), code + 1, code)
    code = code | torch.where(torch.signbit(z), 8, 0)
    code = torch.where(bad.unsqueeze(2), 0, code).reshape(m, k).to(torch.uint8)
    byte = torch.where(bad, 255, (e + 127).to(torch.int64)).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """codes [..., K/2], scale bytes [..., K/32] -> fp64 values [..., K]; scale byte 255 is NaN."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).to(torch.int64)
    s = torch.where(scales == 255, torch.nan, pow2(scales.to(torch.int64) - 127))
    return E2M1.to(codes.device)[c] * s.repeat_interleave(32, dim=-1)


def pack_scales(s: torch.Tensor, fill: int = 127) -> torch.Tensor:
    """Row-major scale bytes [rows, K/32] -> the packed layout: per 128 rows and 128 of K 128 words, word (l, i) <-> row 32 i + l."""
    rows, kb = s.shape
    rp, kp = (rows + 127) // 128 * 128, (kb + 3) // 4 * 4
    full = torch.full((rp, kp), fill, dtype=torch.uint8, device=s.device)
    full[:rows, :kb] = s
    return full.view(rp // 128, 4, 32, kp // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()


def bf16_round(v: torch.Tensor) -> torch.Tensor:
    """fp64 -> nearest bf16 as fp64 (half to even; multiples of 2^-133 in the subnormal range)."""
    _, e = torch.frexp(v)
    step = pow2((e - 8).clamp(-133, 1000))
    return torch.round(v / step) * step


def route(logits: torch.Tensor, top_k: int, scoring="softmax", bias=None, n_group=1, topk_group=1, renormalize=True, scale=1.0):
    """fp64 routing of one token batch; ties go to the lowest index."""
    lg = logits.double()
    score = torch.softmax(lg, dim=1) if scoring == "softmax" else torch.sigmoid(lg)
    pick = score + (bias.double() if bias is not None else 0.0)
    t, e = lg.shape
    if n_group > 1 and topk_group < n_group:
        per = pick.view(t, n_group, e // n_group)
        best = per.sort(dim=2, descending=True).values[:, :, : 2 if bias is not None else 1].sum(dim=2)
        keep = best.sort(dim=1, descending=True, stable=True).indices[:, :topk_group]
        mask = torch.ones(t, n_group, dtype=torch.bool, device=lg.device).scatter_(1, keep, False)
        pick = per.masked_fill(mask.unsqueeze(2), float("-inf")).view(t, e)
    ids = pick.sort(dim=1, descending=True, stable=True).indices[:, :top_k]
    w = score.gather(1, ids)
    if renormalize:
        w = w / w.sum(dim=1, keepdim=True)
    return w * scale, ids


def moe(x, w13, w2, w, ids, fp8_activations=False):
    """fp64 layer and, per output, a bound on the kernel's error.  w13(e), w2(e): the experts' fp64 weights.

    u = 2^-24.  A sum of K fp32 products in any order is off by at most K u sum|a b|.  Beside that the kernel rounds: the
    tokens not at all (bf16 in f16 with a power of two per row), silu's exponential, add and divide and the product with
    the up projection (16 u is generous for the four), the activated rows to 11 bits (2^-11) and the result to bf16 (2^-8).
    |silu'| <= 1.1.
    fp8_activations: the bound of a pipeline that holds gate, up, silu and their product in bf16 (2^-8 each) and rounds tokens and
    activated rows to e4m3 with a power-of-two scale per 128 values: 2^-4 of a value, or half of the smallest step, 2^-10 of a
    scale of at most 2^-7.8 of the largest value (2 / 448), whichever is more."""
    u = 2.0**-24

    def fp8(v):
        return v.abs() * 2.0**-4 + v.abs().amax(dim=1, keepdim=True) * 2.0**-17.8 if fp8_activations else 0.0 * v

    store = 2.0**-8 if fp8_activations else 0.0
    t, h = x.shape
    out = torch.zeros(t, h, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(out)
    for e in ids.unique().tolist():
        tok, slot = (ids == e).nonzero(as_tuple=True)
        a, b = w13(e), w2(e)
        i = a.shape[0] // 2
        xe = x[tok].double()
        both, mag = xe @ a.t(), xe.abs() @ a.abs().t()
        g, up = both[:, :i], both[:, i:]
        d = mag * (h + 16) * u + fp8(xe) @ a.abs().t() + both.abs() * store
        dg, du = d[:, :i], d[:, i:]
        s = g * torch.sigmoid(g)
        y = s * up
        dy = 1.1 * dg * up.abs() + s.abs() * du + 1.1 * dg * du + y.abs() * (16 * u + 2.0**-11 + 2 * store)
        dy = dy + fp8(y.abs() + dy)
        row = y @ b.t()
        drow = dy @ b.abs().t() + (y.abs() @ b.abs().t()) * (i + 16) * u
        ws = w[tok, slot].double().unsqueeze(1)
        out.index_add_(0, tok, ws * row)
        err.index_add_(0, tok, ws.abs() * (drow + row.abs() * (64 * u + store)))      # the weight itself, the weighted sum
    return out, err + out.abs() * 2.0**-8 + 1e-30
