"""The MXFP4 GEMM and linear layer against products in 64 bits: one row to several thousand, ragged N and K, every scheduling
form (weight stream, split K over a cluster, persistent pairs), bias, extreme scales, strides, graphs, and an MLP."""
import pytest
import torch

from tests import mx_reference as ref

pytestmark = pytest.mark.gpu


def operand(rows, k, gen, dev, spread=4):
    q = torch.randint(0, 256, (rows, k // 2), generator=gen, device=dev, dtype=torch.uint8)
    s = torch.randint(127 - spread, 127 + spread, (rows, k // 32), generator=gen, device=dev, dtype=torch.uint8)
    return q, s


def check(got, a, b, bias=None):
    """|error| <= half a bf16 step of the result + the fp32 sum's error: (K + 16) * 2^-22 of the sum of magnitudes.  2^-22, four
    times fp32's half step, because the tensor core adds its products in groups with fewer guard bits than one fp32 add."""
    want = a @ b.t() + (bias.double() if bias is not None else 0.0)
    mag = a.abs() @ b.abs().t() + (bias.double().abs() if bias is not None else 0.0)
    err = want.abs() * 2.0**-8 + mag * (a.shape[1] + 16) * 2.0**-22 + 1e-37
    d = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert float((d / err).max()) <= 1.0


SHAPES = [(1, 8, 32), (1, 1, 128), (3, 24, 160), (9, 17, 64), (16, 256, 256), (77, 2056, 1440), (128, 512, 4096), (129, 300, 544), (200, 4096, 7168),
          (256, 256, 2048), (512, 4096, 7168), (1000, 7168, 2048), (1023, 1000, 96), (2500, 3000, 416), (4096, 5120, 512)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_gemm(cuda_dev, m, n, k, with_bias):
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(m * 7 + n + k)
    aq, asc = operand(m, k, gen, cuda_dev)
    bq, bsc = operand(n, k, gen, cuda_dev)
    bias = torch.randn(n, generator=gen, device=cuda_dev).to(torch.bfloat16) if with_bias else None
    out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device=cuda_dev)
    ops.mxfp4_gemm_nt(aq, ops.pack_mxfp4_scales(asc, k), bq, ops.pack_mxfp4_scales(bsc, k), out, bias)
    check(out, ref.values(aq, asc), ref.values(bq, bsc), bias)
    again = torch.empty_like(out)
    ops.mxfp4_gemm_nt(aq, ops.pack_mxfp4_scales(asc, k), bq, ops.pack_mxfp4_scales(bsc, k), again, bias)
    assert torch.equal(out, again)
    assert ops.gemm_status(cuda_dev) == 0


def linear(x, bq, bsf, n, bias=None, out=None):
    from kb_nano_b200 import ops
    m, k = x.shape
    aq = torch.empty(m, k // 2, dtype=torch.uint8, device=x.device)
    asf = torch.empty(ops.packed_mxfp4_bytes(m, k), dtype=torch.uint8, device=x.device)
    out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device=x.device) if out is None else out
    ops.mxfp4_linear(x, aq, asf, bq, bsf, out, bias)
    return out


@pytest.mark.parametrize("m,n,k", [(1, 4096, 7168), (1, 8, 128), (2, 40, 256), (5, 1, 384), (7, 2056, 1152), (8, 4096, 7168), (8, 24, 8192), (8, 64, 14336), (4, 100, 96),
                                   (9, 512, 512), (33, 136, 1440), (300, 777, 640)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear(cuda_dev, m, n, k, with_bias):
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(m + n + k)
    x = torch.randn(m, k, generator=gen, device=cuda_dev) * torch.exp2(torch.randint(-6, 6, (m, k // 32), generator=gen, device=cuda_dev).float()).repeat_interleave(32, 1)
    x = x.to(torch.bfloat16)
    x[0, :32] = 0
    bq, bsc = operand(n, k, gen, cuda_dev)
    bias = torch.randn(n, generator=gen, device=cuda_dev).to(torch.bfloat16) if with_bias else None
    out = linear(x, bq, ops.pack_mxfp4_scales(bsc, k), n, bias)
    check(out, ref.values(*ref.quant(x)), ref.values(bq, bsc), bias)
    assert ops.gemm_status(cuda_dev) == 0


@pytest.mark.parametrize("m", [2, 40])
def test_scales_at_the_ends_of_the_range(cuda_dev, m):
    """Tiny activations on huge weights and the reverse: results of ordinary size from scales near both ends."""
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(3)
    n, k = 48, 256
    bq, bsc = operand(n, k, gen, cuda_dev)
    for shift in (-90, 90):
        x = (torch.randn(m, k, generator=gen, device=cuda_dev) * 2.0**-shift).to(torch.bfloat16)
        s = (bsc.to(torch.int32) + shift).to(torch.uint8)
        check(linear(x, bq, ops.pack_mxfp4_scales(s, k), n), ref.values(*ref.quant(x)), ref.values(bq, s))


@pytest.mark.parametrize("m", [3, 40])
def test_non_finite_rows_and_weights(cuda_dev, m):
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(4)
    n, k = 64, 256
    bq, bsc = operand(n, k, gen, cuda_dev)
    x = torch.randn(m, k, generator=gen, device=cuda_dev).to(torch.bfloat16)
    clean = linear(x, bq, ops.pack_mxfp4_scales(bsc, k), n)
    x[1, 70] = float("inf")
    bsc[5, 3] = 255
    got = linear(x, bq, ops.pack_mxfp4_scales(bsc, k), n)
    assert torch.isnan(got[1]).all() and torch.isnan(got[:, 5]).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[1] = False
    keep[:, 5] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("m,n", [(3, 72), (40, 72), (300, 1000)])
def test_strided_rows_in_and_out(cuda_dev, m, n):
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(5)
    k = 256
    bq, bsc = operand(n, k, gen, cuda_dev)
    bsf = ops.pack_mxfp4_scales(bsc, k)
    wide = torch.randn(m, k + 13, generator=gen, device=cuda_dev).to(torch.bfloat16)
    for off in (0, 3, 8):
        x = wide[:, off:off + k]
        want = linear(x.contiguous(), bq, bsf, n)
        big = torch.full((m, n + 9), 7.0, dtype=torch.bfloat16, device=cuda_dev)
        linear(x, bq, bsf, n, out=big[:, 4:4 + n])
        assert torch.equal(big[:, 4:4 + n], want) and (big[:, :4] == 7).all() and (big[:, 4 + n:] == 7).all()


def test_weights_written_just_before(cuda_dev):
    """Nothing may be read before the kernel in front has finished: operands, scales and weights made right before the product."""
    from kb_nano_b200 import ops
    m, n, k = 40, 4096, 4096
    gen = torch.Generator(device=cuda_dev).manual_seed(6)
    for rows in (m, 4):
        x = torch.randn(rows, k, generator=gen, device=cuda_dev).to(torch.bfloat16)
        w = torch.randn(2, n, k, generator=gen, device=cuda_dev).to(torch.bfloat16)
        bq = torch.empty(n, k // 2, dtype=torch.uint8, device=cuda_dev)
        bsf = torch.empty(ops.packed_mxfp4_bytes(n, k), dtype=torch.uint8, device=cuda_dev)
        aq = torch.empty(rows, k // 2, dtype=torch.uint8, device=cuda_dev)
        asf = torch.empty(ops.packed_mxfp4_bytes(rows, k), dtype=torch.uint8, device=cuda_dev)
        outs = [[], []]
        for r in range(6):
            o = torch.empty(rows, n, dtype=torch.bfloat16, device=cuda_dev)
            ops.quant_mxfp4(x, aq, packed_sf=asf)
            ops.quant_mxfp4(w[r & 1], bq, packed_sf=bsf)
            if rows > 8:
                ops.mxfp4_gemm_nt(aq, asf, bq, bsf, o)
            else:
                ops.mxfp4_linear(x, aq, asf, bq, bsf, o)
            outs[r & 1].append(o)
        for j in range(2):
            assert all(torch.equal(o, outs[j][0]) for o in outs[j])
            check(outs[j][0], ref.values(*ref.quant(x)), ref.values(*ref.quant(w[j])))


def test_mlp_of_two_linears_and_the_activation_in_a_graph(cuda_dev):
    """quantise -> gate|up product -> SiLU*up and quantise -> down product, eager and replayed, on its own stream."""
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(7)
    h, i = 512, 384
    w13, s13 = operand(2 * i, h, gen, cuda_dev, spread=2)
    w2, s2 = operand(h, i, gen, cuda_dev, spread=2)
    s13 -= 6
    s2 -= 6
    p13, p2 = ops.pack_mxfp4_scales(s13, h), ops.pack_mxfp4_scales(s2, i)
    for m in (1, 8, 100):
        x = torch.randn(m, h, generator=gen, device=cuda_dev).to(torch.bfloat16)
        aq, asf = torch.empty(m, h // 2, dtype=torch.uint8, device=cuda_dev), torch.empty(ops.packed_mxfp4_bytes(m, h), dtype=torch.uint8, device=cuda_dev)
        yq, ysf = torch.empty(m, i // 2, dtype=torch.uint8, device=cuda_dev), torch.empty(ops.packed_mxfp4_bytes(m, i), dtype=torch.uint8, device=cuda_dev)
        ys = torch.empty(m, i // 32, dtype=torch.uint8, device=cuda_dev)
        gu, out = torch.empty(m, 2 * i, dtype=torch.bfloat16, device=cuda_dev), torch.empty(m, h, dtype=torch.bfloat16, device=cuda_dev)

        def mlp():
            ops.mxfp4_linear(x, aq, asf, w13, p13, gu)
            ops.silu_mul_quant_mxfp4(gu, yq, ys, ysf)
            ops.mxfp4_gemm_nt(yq, ysf, w2, p2, out)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            mlp()
        torch.cuda.current_stream().wait_stream(side)
        check(gu, ref.values(*ref.quant(x)), ref.values(w13, s13))
        g, u = gu.double().chunk(2, dim=1)
        cw, sw = ref.quant(ref.bf16_round(ref.bf16_round(g * torch.sigmoid(g)) * u))
        assert torch.equal(yq, cw) and torch.equal(ys, sw)
        check(out, ref.values(yq, ys), ref.values(w2, s2))
        want = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            mlp()
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_no_rows_or_columns(cuda_dev):
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(8)
    bq, bsc = operand(16, 64, gen, cuda_dev)
    assert linear(torch.empty(0, 64, dtype=torch.bfloat16, device=cuda_dev), bq, ops.pack_mxfp4_scales(bsc, 64), 16).shape == (0, 16)
    assert linear(torch.ones(3, 64, dtype=torch.bfloat16, device=cuda_dev), bq[:0], ops.pack_mxfp4_scales(bsc[:0], 64), 0).shape == (3, 0)


def test_refusals(cuda_dev):
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(9)
    m, n, k = 4, 16, 64
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda_dev)
    bq, bsc = operand(n, k, gen, cuda_dev)
    bsf = ops.pack_mxfp4_scales(bsc, k)
    aq, asf = torch.empty(m, k // 2, dtype=torch.uint8, device=cuda_dev), torch.empty(ops.packed_mxfp4_bytes(m, k), dtype=torch.uint8, device=cuda_dev)
    out = torch.empty(m, n, dtype=torch.bfloat16, device=cuda_dev)
    with pytest.raises(ValueError, match="bf16"):
        ops.mxfp4_linear(x.half(), aq, asf, bq, bsf, out)
    with pytest.raises(ValueError, match="b_q"):
        ops.mxfp4_linear(x, aq, asf, bq[:, :16], bsf, out)
    with pytest.raises(ValueError, match="b_sf"):
        ops.mxfp4_linear(x, aq, asf, bq, bsf[:-16], out)
    with pytest.raises(ValueError, match="a_sf"):
        ops.mxfp4_linear(x, aq, asf[16:], bq, bsf, out)
    with pytest.raises(ValueError, match="out must be"):
        ops.mxfp4_linear(x, aq, asf, bq, bsf, out.float())
    with pytest.raises(ValueError, match="bias"):
        ops.mxfp4_linear(x, aq, asf, bq, bsf, out, torch.zeros(n, device=cuda_dev))
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.mxfp4_gemm_nt(aq[:, :24].contiguous(), asf, bq[:, :24].contiguous(), bsf, out)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.mxfp4_gemm_nt(aq.cpu(), asf, bq, bsf, out)


@pytest.mark.parametrize("m", [1, 5, 40])
def test_input_and_output_side_by_side_in_one_matrix(cuda_dev, m):
    """Rows of x and of the result as columns of one buffer: allowed, since they share no memory."""
    from kb_nano_b200 import ops
    n, k = 64, 256
    gen = torch.Generator(device=cuda_dev).manual_seed(60 + m)
    bq, bsc = operand(n, k, gen, cuda_dev)
    bsf = ops.pack_mxfp4_scales(bsc, k)
    both = torch.randn(m, n + k + 8, generator=gen, device=cuda_dev).to(torch.bfloat16)
    before = both.clone()
    want = linear(both[:, n:n + k].contiguous(), bq, bsf, n)
    linear(both[:, n:n + k], bq, bsf, n, out=both[:, :n])
    assert torch.equal(both[:, :n], want) and torch.equal(both[:, n:], before[:, n:])


def test_rows_further_apart_than_32_bit_offsets(cuda_dev):
    """Three rows 1.1 G values apart, in and out of every 4-bit entry point: the same bits as from close rows."""
    from kb_nano_b200 import ops
    ld, k, n = 1_100_000_000, 512, 264
    big = torch.empty(2 * ld + 1024, dtype=torch.bfloat16, device=cuda_dev)
    gen = torch.Generator(device=cuda_dev).manual_seed(70)

    def far(cols, dtype=torch.bfloat16, stride=ld):
        return big.view(dtype).as_strided((3, cols), (stride, 1))

    x = torch.randn(3, k, generator=gen, device=cuda_dev).to(torch.bfloat16)
    q, s = torch.empty(3, k // 2, dtype=torch.uint8, device=cuda_dev), torch.empty(3, k // 32, dtype=torch.uint8, device=cuda_dev)
    sf = torch.empty(ops.packed_mxfp4_bytes(3, k), dtype=torch.uint8, device=cuda_dev)
    ops.quant_mxfp4(x, q, s, sf)
    far(k).copy_(x)
    q2, s2 = torch.empty_like(q), torch.empty_like(s)
    ops.quant_mxfp4(far(k), q2, s2)
    assert torch.equal(q2, q) and torch.equal(s2, s)
    bq, bsc = operand(n, k, gen, cuda_dev)
    bsf = ops.pack_mxfp4_scales(bsc, k)
    want = linear(x, bq, bsf, n)
    assert torch.equal(linear(far(k), bq, bsf, n), want)                                     # far rows in
    linear(x, bq, bsf, n, out=far(n))                                                        # and out, one launch
    assert torch.equal(far(n), want)
    gemm = torch.empty(3, n, dtype=torch.bfloat16, device=cuda_dev)
    ops.mxfp4_gemm_nt(q, sf, bq, bsf, gemm)
    for offset in (0, 3):                                                                    # stored as boxes, and value by value
        view = big.as_strided((3, n), (ld, 1), offset)
        ops.mxfp4_gemm_nt(q, sf, bq, bsf, view)
        assert torch.equal(view, gemm)
    fq, fs = far(k // 2, torch.uint8, 2 * ld - 8), torch.empty_like(s)
    ops.quant_mxfp4(x, fq, fs)
    assert torch.equal(fq, q) and torch.equal(fs, s)
    near = torch.empty_like(x)
    ops.dequant_mxfp4(q, s, near)
    ops.dequant_mxfp4(q, s, far(k))
    assert torch.equal(far(k), near)
    a, b = torch.empty(3, k // 4, dtype=torch.uint8, device=cuda_dev), torch.empty(3, k // 64, dtype=torch.uint8, device=cuda_dev)
    far(k).copy_(x)
    ops.silu_mul_quant_mxfp4(far(k), a, b)
    a2, b2 = torch.empty_like(a), torch.empty_like(b)
    ops.silu_mul_quant_mxfp4(x, a2, b2)
    assert torch.equal(a, a2) and torch.equal(b, b2)
    assert ops.gemm_status(cuda_dev) == 0


FIRST_CALLS = """
import torch
from kb_nano_b200 import moe, ops
d = torch.device("cuda")
torch.manual_seed(0)
k, n = 512, 256
xs = [torch.randn(m, k, device=d).to(torch.bfloat16) for m in (2, 300)]
w = torch.randint(0, 256, (n, k // 2), device=d, dtype=torch.uint8)
wsf = torch.full((ops.packed_mxfp4_bytes(n, k),), 120, dtype=torch.uint8, device=d)
gate = torch.randn(3, 2 * k, device=d).to(torch.bfloat16)
gate[0, :4] = -70.0
lg = torch.randn(2, 4, device=d)
e13, e2 = torch.randint(0, 256, (4, 256, k // 2), device=d, dtype=torch.uint8), torch.randint(0, 256, (4, k, 64), device=d, dtype=torch.uint8)
c13, c2 = torch.full((4, 256, k // 32), 120, dtype=torch.uint8, device=d), torch.full((4, k, 4), 120, dtype=torch.uint8, device=d)
def calls():
    outs = []
    for x in xs:
        m = x.shape[0]
        q, sf = torch.empty(m, k // 2, dtype=torch.uint8, device=d), torch.empty(ops.packed_mxfp4_bytes(m, k), dtype=torch.uint8, device=d)
        outs.append(torch.empty(m, n, dtype=torch.bfloat16, device=d))
        ops.mxfp4_linear(x, q, sf, w, wsf, outs[-1])
    q, s = torch.empty(3, k // 2, dtype=torch.uint8, device=d), torch.empty(3, k // 32, dtype=torch.uint8, device=d)
    ops.silu_mul_quant_mxfp4(gate, q, s)
    outs += [q, s, torch.empty(3, k, dtype=torch.bfloat16, device=d)]
    ops.dequant_mxfp4(q, s, outs[-1])
    outs.append(moe.few_tokens_moe(xs[0], lg, e13, c13, e2, c2, 2))
    return outs
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = calls()
for o in got:
    o.zero_()
g.replay()
want = calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.isfinite(want[0]).all() and ops.gemm_status(d) == 0
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture(cuda_dev):
    import pathlib
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=240, cwd=pathlib.Path(__file__).parents[1])
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_native_calls_accept_what_the_checks_accept(cuda_dev):
    """The native call path takes every well-formed call (whole, strided, on another stream) and turns down one wrong argument at a
    time, whatever it is; the public functions then raise."""
    from kb_nano_b200 import _lib, ops
    calls = _lib.calls()
    m, n, k = 3, 40, 256
    gen = torch.Generator(device=cuda_dev).manual_seed(80)
    wide = torch.randn(m, 2 * k + 6, generator=gen, device=cuda_dev).to(torch.bfloat16)
    x, gu = wide[:, 2:2 + k], wide[:, 4:4 + 2 * k]
    q, s = torch.empty(m, k // 2 + 8, dtype=torch.uint8, device=cuda_dev)[:, :k // 2], torch.empty(m, k // 32 + 3, dtype=torch.uint8, device=cuda_dev)[:, :k // 32]
    p = torch.empty(ops.packed_mxfp4_bytes(m, k), dtype=torch.uint8, device=cuda_dev)
    bq, bsc = operand(n, k, gen, cuda_dev)
    bp, bias = ops.pack_mxfp4_scales(bsc, k), torch.randn(n, generator=gen, device=cuda_dev).to(torch.bfloat16)
    dq, out, back = torch.empty(m, k // 2, dtype=torch.uint8, device=cuda_dev), torch.empty(m, n + 8, dtype=torch.bfloat16, device=cuda_dev)[:, :n], torch.empty_like(x)
    good = [(calls.quant_mxfp4, ops.quant_mxfp4, (x, q, s, p)), (calls.quant_mxfp4, ops.quant_mxfp4, (x, q, None, p)), (calls.quant_mxfp4, ops.quant_mxfp4, (x, dq, s, None)),
            (calls.silu_mul_quant_mxfp4, ops.silu_mul_quant_mxfp4, (gu, q, s, p)), (calls.dequant_mxfp4, ops.dequant_mxfp4, (q, s, back)),
            (calls.mxfp4_gemm_nt, ops.mxfp4_gemm_nt, (dq, p, bq, bp, out, bias)), (calls.mxfp4_linear, ops.mxfp4_linear, (x, dq, p, bq, bp, out, bias)),
            (calls.mxfp4_linear, ops.mxfp4_linear, (x, dq, p, bq, bp, out, None))]
    before = _lib.launch_count()
    for native, public, args in good:
        assert native(*args) is True
        with torch.cuda.stream(torch.cuda.Stream()):
            assert native(*args) is True
        torch.cuda.synchronize()
    assert _lib.launch_count() >= before + 2 * len(good)
    for native, public, args in good:
        for i, a in enumerate(args):
            if a is None:
                continue
            bads = [a.cpu(), a.float(), a[:0], a.t() if a.dim() == 2 else a[: a.numel() - 1], a.double()]
            for bad in bads:
                wrong = (*args[:i], bad, *args[i + 1:])
                if bad.numel() == 0 and i == 0:
                    continue                                      # no rows: nothing to do, not an error
                assert native(*wrong) is False, (native, i, bad.shape, bad.dtype)
                with pytest.raises((ValueError, RuntimeError)):
                    public(*wrong)
    assert ops.gemm_status(cuda_dev) == 0


def test_native_calls_run_on_the_current_stream(cuda_dev):
    """A call inside a stream context is ordered with that stream's work: a long fill before it, a copy behind it."""
    from kb_nano_b200 import ops
    x, y = torch.zeros(4096, 8192, dtype=torch.bfloat16, device=cuda_dev), torch.full((4096, 8192), 3.0, dtype=torch.bfloat16, device=cuda_dev)
    q, s = torch.zeros(4096, 4096, dtype=torch.uint8, device=cuda_dev), torch.zeros(4096, 256, dtype=torch.uint8, device=cuda_dev)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(50):
            x.copy_(y)
            x.mul_(2.0)
        ops.quant_mxfp4(x, q, s)
        got = q.clone(), s.clone()
    stream.synchronize()
    want = ref.quant(torch.full((1, 32), 6.0))
    assert (got[0] == int(want[0][0, 0])).all() and (got[1] == int(want[1][0, 0])).all()


@pytest.mark.parametrize("m", [1, 8, 77, 600])
def test_a_chain_of_launches_equals_the_same_calls_one_by_one(cuda_dev, m):
    """Kernels are let in while the one before them ends.  Thirty rounds over the same buffers, each input the last call's output
    (clamped, since gate * up squares it): the same bits as with a synchronisation after every call."""
    from kb_nano_b200 import ops
    k, n = 512, 1024
    gen = torch.Generator(device=cuda_dev).manual_seed(90 + m)
    bq, bsc = operand(n, k, gen, cuda_dev, 2)
    bsf = ops.pack_mxfp4_scales((bsc - 4), k)
    start = torch.randn(m, k, generator=gen, device=cuda_dev).to(torch.bfloat16)

    def chain(wait):
        x, q, s = start.clone(), torch.empty(m, k // 2, dtype=torch.uint8, device=cuda_dev), torch.empty(m, k // 32, dtype=torch.uint8, device=cuda_dev)
        aq, asf = torch.empty_like(q), torch.empty(ops.packed_mxfp4_bytes(m, k), dtype=torch.uint8, device=cuda_dev)
        y, seen = torch.empty(m, n, dtype=torch.bfloat16, device=cuda_dev), []
        torch.cuda.synchronize()
        for i in range(30):
            for f in (lambda: ops.mxfp4_linear(x, aq, asf, bq, bsf, y), lambda: ops.silu_mul_quant_mxfp4(y, q, s), lambda: ops.dequant_mxfp4(q, s, x),
                      lambda: x.clamp_(-1, 1).add_(start), lambda: ops.quant_mxfp4(x, q, s), lambda: ops.dequant_mxfp4(q, s, x)):
                f()
                if wait:
                    torch.cuda.synchronize()
            seen.append((x.clone(), q.clone(), s.clone()))
        torch.cuda.synchronize()
        return seen

    want = chain(True)
    assert all(torch.isfinite(a[0]).all() for a in want) and not torch.equal(want[0][0], want[-1][0])
    for _ in range(5):
        got = chain(False)
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@pytest.mark.parametrize("m,n,k", [(300, 2600, 9216), (512, 4608, 9280), (257, 2561, 9984), (77, 2056, 12320), (1, 1000, 16384), (40, 8, 14336)])
def test_gemm_with_k_split_over_a_cluster(cuda_dev, m, n, k):
    """Few tiles and long K, two and four slices, whole boxes and ragged edges."""
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(m + n + k)
    aq, asc = operand(m, k, gen, cuda_dev)
    bq, bsc = operand(n, k, gen, cuda_dev)
    bias = torch.randn(n, generator=gen, device=cuda_dev).to(torch.bfloat16)
    asf, bsf = ops.pack_mxfp4_scales(asc, k), ops.pack_mxfp4_scales(bsc, k)
    a, b = ref.values(aq, asc), ref.values(bq, bsc)
    for bb in (None, bias):
        out, again = torch.full((m, n + 8), 7.0, dtype=torch.bfloat16, device=cuda_dev), torch.empty(m, n, dtype=torch.bfloat16, device=cuda_dev)
        ops.mxfp4_gemm_nt(aq, asf, bq, bsf, out[:, :n], bb)
        check(out[:, :n], a, b, bb)
        assert (out[:, n:] == 7).all()
        ops.mxfp4_gemm_nt(aq, asf, bq, bsf, again, bb)
        assert torch.equal(out[:, :n], again)
    assert ops.gemm_status(cuda_dev) == 0


@pytest.mark.parametrize("m,n,k,pad", [(1280, 4096, 512, 8), (1270, 4200, 544, 8), (1270, 4200, 544, 3), (2304, 2309, 96, 0), (300, 12800, 2080, 8)])
def test_gemm_with_a_halved_last_round(cuda_dev, m, n, k, pad):
    """A few tiles more than pairs: the last round's tiles in halves, of which the outer may lie behind the last column."""
    from kb_nano_b200 import ops
    gen = torch.Generator(device=cuda_dev).manual_seed(m + n + k + pad)
    aq, asc = operand(m, k, gen, cuda_dev)
    bq, bsc = operand(n, k, gen, cuda_dev)
    bias = torch.randn(n, generator=gen, device=cuda_dev).to(torch.bfloat16)
    asf, bsf = ops.pack_mxfp4_scales(asc, k), ops.pack_mxfp4_scales(bsc, k)
    a, b = ref.values(aq, asc), ref.values(bq, bsc)
    for bb in (None, bias):
        buf = torch.full((m + 1, n + pad), 7.0, dtype=torch.bfloat16, device=cuda_dev)
        out = buf[:m, :n]
        ops.mxfp4_gemm_nt(aq, asf, bq, bsf, out, bb)
        check(out, a, b, bb)
        assert (buf[m] == 7).all() and (buf[:, n:] == 7).all()
    assert ops.gemm_status(cuda_dev) == 0
