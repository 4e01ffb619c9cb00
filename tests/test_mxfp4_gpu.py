"""MXFP4 quantisers against their definition in 64 bits: codes, scale bytes and the packed layout are bit-exact; every bf16
magnitude, odd sizes, strides, infinities and NaNs, the fused activation over every gate, the inverse."""
import pytest
import torch

from tests import mx_reference as ref

pytestmark = pytest.mark.gpu


def outputs(m, k, dev):
    from kb_nano_b200 import ops
    return (torch.full((m, k // 2), 0xEE, dtype=torch.uint8, device=dev), torch.full((m, k // 32), 0xEE, dtype=torch.uint8, device=dev),
            torch.full((ops.packed_mxfp4_bytes(m, k),), 0xEE, dtype=torch.uint8, device=dev))


def check_packed(got, scales):
    """Written words equal the packed row-major scales; words of rows past the last one are left alone."""
    rows, kb = scales.shape
    want = ref.pack_scales(scales).view(-1, 128, 4)
    row = (torch.arange(128, device=scales.device) // 4 + 32 * (torch.arange(128, device=scales.device) % 4)).repeat(want.shape[0], 1)
    row = row + (torch.arange(want.shape[0], device=scales.device) // ((kb + 3) // 4)).unsqueeze(1) * 128
    g = got.view(-1, 128, 4)
    assert torch.equal(g[row < rows], want[row < rows])
    assert (g[row >= rows] == 0xEE).all()


def check_quant(x, codes, scales, packed):
    cw, sw = ref.quant(x)
    assert torch.equal(scales, sw) and torch.equal(codes, cw)
    check_packed(packed, sw)


@pytest.mark.parametrize("m,k", [(1, 32), (1, 7168), (3, 64), (127, 96), (128, 128), (129, 160), (200, 1440), (512, 2048), (1000, 544)])
def test_quant(cuda_dev, m, k):
    from kb_nano_b200 import ops
    x = torch.randn(m, k, device=cuda_dev) * torch.exp2(torch.randint(-12, 12, (m, k // 32), device=cuda_dev).float()).repeat_interleave(32, dim=1)
    x = x.to(torch.bfloat16)
    x[0, :32] = 0
    q, s, p = outputs(m, k, cuda_dev)
    ops.quant_mxfp4(x, q, s, p)
    check_quant(x, q, s, p)
    q2, s2, p2 = outputs(m, k, cuda_dev)
    ops.quant_mxfp4(x, q2, out_scale=s2)                                  # each place for the scales alone
    assert torch.equal(q2, q) and torch.equal(s2, s)
    ops.quant_mxfp4(x, q2, packed_sf=p2)
    assert torch.equal(p2, p)
    assert torch.equal(ops.pack_mxfp4_scales(s, k), ref.pack_scales(s))


def test_every_bf16_value_as_block_maximum_and_as_element(cuda_dev):
    """All 65,536 bit patterns: each as the largest of a block, beside a spread of values below it."""
    from kb_nano_b200 import ops
    bits = torch.arange(65536, device=cuda_dev, dtype=torch.int32).to(torch.int16)
    top = bits.view(torch.bfloat16)
    frac = torch.linspace(0, 1, 31, device=cuda_dev)
    x = torch.cat([top.unsqueeze(1), (top.float().unsqueeze(1) * frac).to(torch.bfloat16)], dim=1).view(512, 128 * 32)
    q, s, p = outputs(512, 4096, cuda_dev)
    ops.quant_mxfp4(x, q, s, p)
    check_quant(x, q, s, p)


def test_midpoints_round_to_even_codes(cuda_dev):
    from kb_nano_b200 import ops
    v = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -6.0] * 2, device=cuda_dev)
    x = torch.stack([v * 2.0**e for e in (-20, -1, 0, 3, 40)]).to(torch.bfloat16)
    q, s, p = outputs(5, 32, cuda_dev)
    ops.quant_mxfp4(x, q, s, p)
    check_quant(x, q, s, p)
    back = torch.empty_like(x)
    ops.dequant_mxfp4(q, s, back)
    assert back[2].tolist()[:8] == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]


def test_infinities_and_nans_spoil_their_block_only(cuda_dev):
    from kb_nano_b200 import ops
    x = torch.randn(4, 256, device=cuda_dev).to(torch.bfloat16)
    x[0, 5], x[1, 64], x[2, 255], x[3, 40] = float("nan"), float("inf"), float("-inf"), float("nan")
    q, s, p = outputs(4, 256, cuda_dev)
    ops.quant_mxfp4(x, q, s, p)
    check_quant(x, q, s, p)
    back = torch.empty_like(x)
    ops.dequant_mxfp4(q, s, back)
    bad = torch.isnan(back).view(4, 8, 32)
    want = torch.zeros(4, 8, dtype=torch.bool, device=cuda_dev)
    want[0, 0] = want[1, 2] = want[2, 7] = want[3, 1] = True
    assert torch.equal(bad.all(dim=2), want) and torch.equal(bad.any(dim=2), want)


@pytest.mark.parametrize("off,ld", [(0, 200), (1, 201), (3, 260), (8, 264)])
def test_strides_and_alignment(cuda_dev, off, ld):
    from kb_nano_b200 import ops
    m, k = 37, 192
    wide = torch.randn(m, ld, device=cuda_dev).to(torch.bfloat16)
    x = torch.as_strided(wide, (m, k), (ld, 1), off) if off + k <= ld else wide[:, :k]
    qw = torch.full((m, k // 2 + 20), 0xEE, dtype=torch.uint8, device=cuda_dev)
    sw = torch.full((m, k // 32 + 3), 0xEE, dtype=torch.uint8, device=cuda_dev)
    q, s = qw[:, 4:4 + k // 2], sw[:, 1:1 + k // 32]
    ops.quant_mxfp4(x, q, s)
    cw, scw = ref.quant(x)
    assert torch.equal(q, cw) and torch.equal(s, scw)
    assert (qw[:, :4] == 0xEE).all() and (qw[:, 4 + k // 2:] == 0xEE).all() and (sw[:, 0] == 0xEE).all() and (sw[:, 1 + k // 32:] == 0xEE).all()
    assert torch.equal(ops.pack_mxfp4_scales(s, k), ref.pack_scales(scw))
    ow = torch.full((m, ld), 7.0, dtype=torch.bfloat16, device=cuda_dev)
    o = torch.as_strided(ow, (m, k), (ld, 1), off) if off + k <= ld else ow[:, :k]
    ops.dequant_mxfp4(q, s, o)
    assert torch.equal(o.double(), ref.values(cw, scw))
    first = off if off + k <= ld else 0
    keep = torch.ones(ld, dtype=torch.bool, device=cuda_dev)
    keep[first:first + k] = False
    assert (ow[:, keep] == 7).all()


def test_dequant_every_code_under_every_scale(cuda_dev):
    from kb_nano_b200 import ops
    q = torch.arange(256, dtype=torch.uint8, device=cuda_dev).repeat(256, 1)
    s = torch.arange(256, dtype=torch.uint8, device=cuda_dev).unsqueeze(1).repeat(1, 16)
    out = torch.empty(256, 512, dtype=torch.bfloat16, device=cuda_dev)
    ops.dequant_mxfp4(q, s, out)
    want = ref.values(q, s).float().to(torch.bfloat16)
    assert torch.equal(out.view(torch.int16)[s[:, 0] != 255], want.view(torch.int16)[s[:, 0] != 255])
    assert torch.isnan(out[255]).all()


@pytest.mark.parametrize("m,n", [(1, 32), (129, 2048), (77, 96), (5, 1440), (700, 544)])
def test_silu_mul_quant(cuda_dev, m, n):
    from kb_nano_b200 import ops
    x = (torch.randn(m, 2 * n, device=cuda_dev) * 3).to(torch.bfloat16)
    q, s, p = outputs(m, n, cuda_dev)
    ops.silu_mul_quant_mxfp4(x, q, s, p)
    g, u = x.double().chunk(2, dim=1)
    check_quant(ref.bf16_round(ref.bf16_round(g * torch.sigmoid(g)) * u), q, s, p)


def test_silu_mul_quant_over_every_finite_gate(cuda_dev):
    """Every finite gate in bf16's normal range, up = 1.5 (a product that rounds), in blocks of neighbouring values."""
    from kb_nano_b200 import ops
    bits = torch.arange(65536, device=cuda_dev, dtype=torch.int32)
    mag = bits & 0x7FFF
    gate = torch.where((mag >= 0x80) & (mag < 0x7F80) & ~((bits >= 0x8000) & (mag > 0x42A0)), bits, 0x3F80).to(torch.int16).view(torch.bfloat16).view(64, 1024)
    x = torch.cat([gate, torch.full_like(gate, 1.5)], dim=1)
    q, s, p = outputs(64, 1024, cuda_dev)
    ops.silu_mul_quant_mxfp4(x, q, s, p)
    g = gate.double()
    y = ref.bf16_round(ref.bf16_round(g / (1 + torch.exp(-g))) * 1.5)
    y = torch.where(y.abs() >= 2.0**128, torch.inf, y)
    check_quant(y, q, s, p)


def test_silu_of_gates_far_below_zero_and_non_finite(cuda_dev):
    """Gates below -60 beside ordinary ones; infinities and NaNs spoil their block."""
    from kb_nano_b200 import ops
    x = torch.randn(8, 128, device=cuda_dev).to(torch.bfloat16)
    x[0, 3], x[1, 9], x[2, 33] = -60.5, -87.5, -88.0
    x[3, 2], x[4, 5], x[5, 63], x[6, 100] = float("nan"), float("inf"), float("-inf"), float("nan")
    q, s, p = outputs(8, 64, cuda_dev)
    ops.silu_mul_quant_mxfp4(x, q, s, p)
    g, u = x.double().chunk(2, dim=1)
    check_quant(ref.bf16_round(ref.bf16_round(torch.where(torch.isinf(g) & (g < 0), torch.nan, g * torch.sigmoid(g))) * u), q, s, p)


def test_silu_strides(cuda_dev):
    from kb_nano_b200 import ops
    wide = torch.randn(9, 140, device=cuda_dev).to(torch.bfloat16)
    for off in (0, 3, 8):
        x = wide[:, off:off + 128]
        q, s, p = outputs(9, 64, cuda_dev)
        ops.silu_mul_quant_mxfp4(x, q, s, p)
        q2, s2, p2 = outputs(9, 64, cuda_dev)
        ops.silu_mul_quant_mxfp4(x.contiguous(), q2, s2, p2)
        assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(p, p2)


def test_no_rows(cuda_dev):
    from kb_nano_b200 import ops
    q, s, _ = outputs(0, 64, cuda_dev)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=cuda_dev)
    ops.quant_mxfp4(x, q, s)
    ops.dequant_mxfp4(q, s, x)
    ops.silu_mul_quant_mxfp4(torch.empty(0, 128, dtype=torch.bfloat16, device=cuda_dev), q, s)
    assert ops.pack_mxfp4_scales(s, 64).numel() == 0


def test_other_dtypes_of_codes_and_scales(cuda_dev):
    from kb_nano_b200 import ops
    x = torch.randn(8, 128, device=cuda_dev).to(torch.bfloat16)
    q, s, _ = outputs(8, 128, cuda_dev)
    ops.quant_mxfp4(x, q, s)
    q2, s2, _ = outputs(8, 128, cuda_dev)
    ops.quant_mxfp4(x, q2.view(torch.float4_e2m1fn_x2), s2.view(torch.float8_e8m0fnu))
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_quant_refusals(cuda_dev):
    from kb_nano_b200 import ops
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda_dev)
    q, s, p = outputs(4, 64, cuda_dev)
    with pytest.raises(ValueError, match="bf16"):
        ops.quant_mxfp4(x.float(), q, s)
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.quant_mxfp4(x[:, :48], q[:, :24], s)
    with pytest.raises(ValueError, match="out_fp4"):
        ops.quant_mxfp4(x, q[:, :16], s)
    with pytest.raises(ValueError, match="out_scale"):
        ops.quant_mxfp4(x, q, s.float())
    with pytest.raises(ValueError, match="packed_sf"):
        ops.quant_mxfp4(x, q, None, p[:-1])
    with pytest.raises(ValueError, match="give out_scale"):
        ops.quant_mxfp4(x, q)
    with pytest.raises(ValueError, match="contiguous along"):
        ops.quant_mxfp4(torch.zeros(64, 4, dtype=torch.bfloat16, device=cuda_dev).t(), q, s)
    with pytest.raises(RuntimeError, match="4-byte"):
        ops.quant_mxfp4(x, torch.zeros(4, 33, dtype=torch.uint8, device=cuda_dev)[:, :32], s)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.quant_mxfp4(x.cpu(), q.cpu(), s.cpu())
    with pytest.raises(ValueError, match="out must be"):
        ops.dequant_mxfp4(q, s, x.float())
