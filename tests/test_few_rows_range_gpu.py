"""Few-row kernels (mxfp4_linear on up to eight rows, few_tokens_moe) over the range of their types: powers of two that tokens
and weight scales take from each other, blocks of very different size side by side, sums that cancel.  Every case is built so
that the results are of ordinary size and a value lost on the way shows in them."""
import pytest
import torch

from tests import mx_reference as ref
from tests.test_moe_few_gpu import FP8, experts
from tests.test_mxfp4_gemm_gpu import check, linear, operand

pytestmark = pytest.mark.gpu
U = 2.0**-24


def moe_bounds(x, w13, w2, w, ids, n13=None, n2=None, row=2.0**-11):
    """The layer in 64 bits and a bound on an evaluation that rounds to fp32 at every step and to bf16 once, at the end.

    A sum of n fp32 products other than zero (n13, n2: at most that many a row) in any order is off by at most n u sum|a b|
    (u = 2^-24); scales and powers of two add a few more roundings, 16 u in all.  silu's exponential, add and divide and the product with the up projection: 16 u; the
    activated rows' own rounding, `row` of the value (f16: 2^-11) or, where a value is far below its block's largest, half of f16's
    smallest step (2^-25) beside a largest of at least 2^14: 2^-39 of the largest of at most 128.  |silu'| <= 1.1."""
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
        d = mag * ((n13 or h) + 16) * U
        dg, du = d[:, :i], d[:, i:]
        s = g * torch.sigmoid(g)
        y = s * up
        dy = 1.1 * dg * up.abs() + s.abs() * du + 1.1 * dg * du + y.abs() * (16 * U + row)
        dy = dy + (y.abs() + dy).view(len(tok), -1, 128).amax(dim=2).repeat_interleave(128, dim=1) * 2.0**-39
        drow = dy @ b.abs().t() + (y.abs() @ b.abs().t()) * ((n2 or i) + 16) * U
        ws = w[tok, slot].double().unsqueeze(1)
        out.index_add_(0, tok, ws * (y @ b.t()))
        err.index_add_(0, tok, ws.abs() * (drow + (y @ b.t()).abs() * 64 * U))      # the weight itself, the weighted sum
    return out, err + out.abs() * 2.0**-8 + 1e-38


def check_moe(dev, x, logits, ex, top=2, **bound):
    from kb_nano_b200 import moe, ops
    w13, s13, w2, s2, f13, f2 = ex
    got = moe.few_tokens_moe(x, logits, w13, s13, w2, s2, top)
    w, ids = ref.route(logits, top)
    want, err = moe_bounds(x, f13, f2, w, ids, **bound)
    assert torch.isfinite(want).all() and torch.isfinite(got).all()
    assert float(want.abs().max()) > 1e-6                              # of ordinary size: nothing hides below the bound
    worst = float(((got.double() - want).abs() / err).max())
    assert worst <= 1.0, f"error {worst:.3g} times its bound"
    assert ops.gemm_status(dev) == 0


def shifted(fmt, e, h, i, dev, seed, by13, by2):
    """Experts whose weight scales carry 2^by13 and 2^by2."""
    w13, s13, w2, s2, _, _ = experts(fmt, e, h, i, dev, seed)
    if fmt == "fp8":
        s13, s2 = s13 * 2.0**by13, s2 * 2.0**by2
        return w13, s13, w2, s2, *(lambda x, q=q, s=s: q[x].double() * s[x].double().repeat_interleave(128, 0).repeat_interleave(128, 1) for q, s in ((w13, s13), (w2, s2)))
    s13, s2 = (s13.int() + by13).clamp(0, 254).to(torch.uint8), (s2.int() + by2).clamp(0, 254).to(torch.uint8)
    return w13, s13, w2, s2, *(lambda x, q=q, s=s: ref.values(q[x], s[x]) for q, s in ((w13, s13), (w2, s2)))


@pytest.mark.parametrize("m", [1, 2, 8, 9, 40])
@pytest.mark.parametrize("shift", [-120, -110, 100, 115, 120])
def test_linear_scales_near_both_ends_of_the_range(cuda_dev, m, shift):
    """Activations of 2^-shift on weight scales of 2^shift: the kernels of one to eight and of more rows alike."""
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(100 + m)
    n, k = 48, 512
    bq, bsc = operand(n, k, gen, cuda_dev)
    x = (torch.randn(m, k, generator=gen, device=cuda_dev) * 2.0**-shift).to(torch.bfloat16)
    s = (bsc.to(torch.int32) + shift).to(torch.uint8)
    check(linear(x, bq, ops.pack_mxfp4_scales(s, k), n), ref.values(*ref.quant(x)), ref.values(bq, s))


@pytest.mark.parametrize("m", [8, 9])
@pytest.mark.parametrize("apart", [30, 40, 70])
def test_linear_blocks_far_apart_within_128_values(cuda_dev, m, apart):
    """Neighbouring blocks of 32 up to 2^210 apart, their weights' scales the other way round: every block counts alike."""
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(200 + m + apart)
    n, k = 40, 384
    power = ((torch.arange(k // 32, device=cuda_dev) % 4) - 1) * apart
    power = power.clamp(-100, 100)
    bq, bsc = operand(n, k, gen, cuda_dev)
    x = (torch.randn(m, k, generator=gen, device=cuda_dev) * torch.exp2(power.float()).repeat_interleave(32)).to(torch.bfloat16)
    s = (bsc.to(torch.int32) - power).to(torch.uint8)
    check(linear(x, bq, ops.pack_mxfp4_scales(s, k), n), ref.values(*ref.quant(x)), ref.values(bq, s))


@pytest.mark.parametrize("m", [3, 20])
def test_linear_empty_weight_blocks_of_any_scale(cuda_dev, m):
    """A block without a value contributes nothing, whatever its scale byte says and however large the activations are."""
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(300 + m)
    n, k = 40, 256
    bq, bsc = operand(n, k, gen, cuda_dev)
    x = torch.randn(m, k, generator=gen, device=cuda_dev)
    x[:, 32:64] *= 2.0**100
    x = x.to(torch.bfloat16)
    bq[:, 16:32] = 0
    bsc[:, 1] = 254
    check(linear(x, bq, ops.pack_mxfp4_scales(bsc, k), n), ref.values(*ref.quant(x)), ref.values(bq, bsc))


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t", [1, 5, 16])
@pytest.mark.parametrize("shift", [-118, -90, 90, 120])
def test_moe_tokens_against_weight_scales(cuda_dev, fmt, t, shift):
    """Tokens of 2^-shift, gate and up scales of 2^shift: gate, up and the result of order one."""
    gen = torch.Generator(device=cuda_dev).manual_seed(400 + t)
    x = (torch.randn(t, 256, generator=gen, device=cuda_dev) * 2.0**-shift).to(torch.bfloat16)
    lg = torch.randn(t, 4, generator=gen, device=cuda_dev)
    check_moe(cuda_dev, x, lg, shifted(fmt, 4, 256, 256, cuda_dev, 41, shift, 0))


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t", [2, 16])
@pytest.mark.parametrize("by13", [-58, -40, 40, 58])
def test_moe_activated_rows_against_weight_scales(cuda_dev, fmt, t, by13):
    """Gate and up of 2^by13 each, so activated rows of about 2^(2 by13), and down scales that take it out again."""
    gen = torch.Generator(device=cuda_dev).manual_seed(500 + t)
    x = torch.randn(t, 256, generator=gen, device=cuda_dev).to(torch.bfloat16)
    lg = torch.randn(t, 4, generator=gen, device=cuda_dev)
    check_moe(cuda_dev, x, lg, shifted(fmt, 4, 256, 256, cuda_dev, 42, by13, -2 * by13))


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_moe_small_values_beside_large_ones(cuda_dev, fmt):
    """Every other token value 2^25 times the ones between, the large ones' weights zero: the small ones are what counts."""
    gen = torch.Generator(device=cuda_dev).manual_seed(600)
    w13, s13, w2, s2, f13, f2 = shifted(fmt, 4, 256, 128, cuda_dev, 43, 25, 0)
    if fmt == "fp8":
        w13.view(torch.uint8)[:, :, 0::2] = 0
    else:
        w13 &= 0xF0
    x = torch.randn(6, 256, generator=gen, device=cuda_dev)
    x[:, 1::2] *= 2.0**-25
    lg = torch.randn(6, 4, generator=gen, device=cuda_dev)
    check_moe(cuda_dev, x.to(torch.bfloat16), lg, (w13, s13, w2, s2, f13, f2))


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,e", [(1, 4), (3, 4), (4, 2), (5, 2), (8, 2), (16, 2)])
@pytest.mark.parametrize("i", [256, 1280, 7424])
def test_moe_activated_rows_keep_more_than_f16(cuda_dev, fmt, t, e, i):
    """Neighbouring activated values that differ by 2^-13 and the down projection's difference of the two: what is left of
    them is the result, and rounding them to 11 bits would be most of it.  One to eight tokens an expert and more."""
    gen = torch.Generator(device=cuda_dev).manual_seed(700 + t)
    h = 256
    w13, s13, w2, s2, f13, f2 = shifted(fmt, e, h, i, cuda_dev, 44, 0, 17)
    x = torch.zeros(t, h, device=cuda_dev)                              # two values a row, so that the sums round little
    x[:, 0] = torch.randn(t, generator=gen, device=cuda_dev)
    x[:, h - 1] = torch.randn(t, generator=gen, device=cuda_dev) * 2.0**-13
    b13, b2 = w13.view(torch.uint8), w2.view(torch.uint8)
    # gate rows 2j and 2j + 1 alike; up rows too but for the last value; four down columns, neighbours of opposite sign
    b13[:, 1::2] = b13[:, 0::2]
    if fmt == "fp8":
        b13[:, :, h - 1] = 0
        b13[:, i + 1::2, h - 1] = 0x74                                    # 192
        b2[:, :, 2:i - 2] = 0
        b2[:, :, 1::2] = b2[:, :, 0::2] ^ 0x80
    else:
        s13[:, 1::2] = s13[:, 0::2]
        b13[:, :, h // 2 - 1] &= 0x0F
        b13[:, i + 1::2, h // 2 - 1] |= 0x70                              # 6
        b2[:, :, 1:i // 2 - 1] = 0
        b2 &= 0x0F
        b2 |= (b2 << 4) ^ 0x80
    lg = torch.randn(t, e, generator=gen, device=cuda_dev)
    check_moe(cuda_dev, x.to(torch.bfloat16), lg, (w13, s13, w2, s2, f13, f2), top=1 if t > 8 else 2, n13=2, n2=4, row=2.0**-22)


@pytest.mark.parametrize("fmt,h", [("fp8", 74624), ("mxfp4", 62848)])
@pytest.mark.parametrize("t", [1, 16])
def test_moe_longest_token_rows(cuda_dev, fmt, h, t):
    """The largest H that is taken: one token at a time beside a ring of three stages."""
    from kb_nano_b200 import moe
    gen = torch.Generator(device=cuda_dev).manual_seed(800 + t)
    x = torch.randn(t, h, generator=gen, device=cuda_dev).to(torch.bfloat16)
    lg = torch.randn(t, 2, generator=gen, device=cuda_dev)
    ex = experts(fmt, 2, h, 128, cuda_dev, 45)
    check_moe(cuda_dev, x, lg, ex, top=1)
    with pytest.raises(RuntimeError, match="shared memory"):
        longer = torch.cat([x, x[:, :128]], dim=1)
        moe.few_tokens_moe(longer, lg, *experts(fmt, 2, h + 128, 128, cuda_dev, 46)[:4], 1)
