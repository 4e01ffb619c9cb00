"""The MoE layer for a few tokens (moe.few_tokens_moe) against the layer in 64 bits: FP8 and MXFP4 experts, 1 to 16 tokens,
odd sizes, all routings; one expert for every token, non-finite inputs, strides, streams, captured graphs, refusals."""
import pytest
import torch

from tests import mx_reference as ref

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def experts(fmt, e, h, i, dev, seed):
    """(w13, s13, w2, s2, fp64 weight of expert x as functions)."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for n, k in ((2 * i, h), (h, i)):
        if fmt == "fp8":
            q = (torch.randn(e, n, k, generator=gen, device=dev) * 100.0).clamp(-448, 448).to(FP8)
            s = torch.rand(e, n // 128, k // 128, generator=gen, device=dev) * 2e-4 + 1e-4
        else:
            q = torch.randint(0, 256, (e, n, k // 2), generator=gen, device=dev, dtype=torch.uint8)
            s = torch.randint(116, 123, (e, n, k // 32), generator=gen, device=dev, dtype=torch.uint8)
        out += [q, s]
    if fmt == "fp8":
        def val(q, s):
            return lambda x: q[x].double() * s[x].double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    else:
        def val(q, s):
            return lambda x: ref.values(q[x], s[x])
    return (*out, val(out[0], out[1]), val(out[2], out[3]))


def check(got, want, err):
    d = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    worst = float((d / err).max())
    assert worst <= 1.0, f"error {worst:.3g} times its bound"


def run_case(dev, fmt, t, h, i, e, top, seed=0, logits=None, x=None, dtype=torch.float32, **route):
    from kb_nano_b200 import moe
    gen = torch.Generator(device=dev).manual_seed(1000 + seed)
    w13, s13, w2, s2, f13, f2 = experts(fmt, e, h, i, dev, seed)
    x = torch.randn(t, h, generator=gen, device=dev).to(torch.bfloat16) if x is None else x
    logits = torch.randn(t, e, generator=gen, device=dev).to(dtype) if logits is None else logits
    ow, oi = torch.empty(t, top, device=dev), torch.empty(t, top, dtype=torch.int32, device=dev)
    got = moe.few_tokens_moe(x, logits, w13, s13, w2, s2, top, out_w=ow, out_ids=oi, **route)
    w, ids = ref.route(logits, top, **route)
    assert torch.equal(oi.long(), ids)
    # expf, the sum over E scores, the division: 64 u is generous
    assert float(((ow.double() - w).abs() / w.clamp_min(1e-300)).max()) <= (64 + e) * 2.0**-24
    check(got, *ref.moe(x, f13, f2, w, ids))
    return got


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,h,i,e,top", [(1, 128, 128, 1, 1), (1, 2048, 768, 128, 8), (2, 256, 128, 4, 2), (3, 384, 640, 9, 3), (7, 1152, 1408, 16, 4),
                                         (8, 512, 256, 8, 8), (9, 512, 256, 8, 8), (16, 1024, 512, 64, 8), (16, 256, 384, 2, 1), (16, 640, 128, 300, 16),
                                         (5, 128, 14336, 3, 2), (4, 7168, 2048, 8, 2), (11, 16384, 128, 3, 2),
                                         # rows of 7168 for eight tokens leave the FP8 ring an odd number of stages
                                         (8, 7168, 256, 8, 4), (16, 7168, 2048, 24, 8), (13, 6656, 512, 16, 6)])
def test_matches_the_layer_in_64_bits(cuda_dev, fmt, t, h, i, e, top):
    run_case(cuda_dev, fmt, t, h, i, e, top, seed=t + h)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_grouped_sigmoid_routing_with_bias(cuda_dev, fmt):
    bias = torch.randn(64, device=cuda_dev) * 0.1
    run_case(cuda_dev, fmt, 6, 512, 256, 64, 4, seed=5, scoring="sigmoid", bias=bias, n_group=8, topk_group=3, scale=2.5)


def test_bf16_logits_and_ties(cuda_dev):
    lg = torch.zeros(4, 32, device=cuda_dev, dtype=torch.bfloat16)        # all equal: the lowest indices win
    run_case(cuda_dev, "fp8", 4, 256, 128, 32, 4, seed=6, logits=lg)
    run_case(cuda_dev, "fp8", 4, 256, 128, 32, 4, seed=7, dtype=torch.bfloat16)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_every_token_on_the_same_experts(cuda_dev, fmt):
    lg = torch.full((16, 8), -20.0, device=cuda_dev)
    lg[:, 3], lg[:, 5] = 4.0, 3.0
    run_case(cuda_dev, fmt, 16, 512, 256, 8, 2, seed=8, logits=lg)


def test_experts_masked_out_with_minus_infinity(cuda_dev):
    lg = torch.randn(3, 16, device=cuda_dev)
    lg[:, 4:] = float("-inf")
    run_case(cuda_dev, "fp8", 3, 256, 128, 16, 4, seed=9, logits=lg)


@pytest.mark.parametrize("factor", [1e-30, 2.0**-100, 1e4])
def test_tokens_far_from_one(cuda_dev, factor):
    """Rows of very different magnitude in one call; the per-row power of two keeps each exact."""
    x = torch.randn(4, 512, device=cuda_dev).to(torch.bfloat16)
    x[1] *= factor
    x[2] = 0
    run_case(cuda_dev, "fp8", 4, 512, 256, 8, 2, seed=10, x=x)


def test_non_finite_tokens_stay_in_their_row(cuda_dev):
    from kb_nano_b200 import moe
    w13, s13, w2, s2, _, _ = experts("fp8", 8, 256, 128, cuda_dev, 11)
    x = torch.randn(5, 256, device=cuda_dev).to(torch.bfloat16)
    lg = torch.randn(5, 8, device=cuda_dev)
    clean = moe.few_tokens_moe(x, lg, w13, s13, w2, s2, 2)
    x[1, 7], x[3, 100] = float("nan"), float("inf")
    lg[4, 2] = float("nan")
    ids = torch.empty(5, 2, dtype=torch.int32, device=cuda_dev)
    got = moe.few_tokens_moe(x, lg, w13, s13, w2, s2, 2, out_w=torch.empty(5, 2, device=cuda_dev), out_ids=ids)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    assert torch.isnan(got[1]).all() and not torch.isfinite(got[3]).any() and torch.isnan(got[4]).all()
    assert (ids[4] == -1).all()
    lg[:] = float("nan")                                                 # no token has an expert
    assert torch.isnan(moe.few_tokens_moe(x, lg, w13, s13, w2, s2, 2)).all()


def test_strided_rows_and_in_place_output(cuda_dev):
    from kb_nano_b200 import moe
    w13, s13, w2, s2, _, _ = experts("mxfp4", 8, 256, 128, cuda_dev, 12)
    wide = torch.randn(6, 512, device=cuda_dev).to(torch.bfloat16)
    lgw = torch.randn(6, 20, device=cuda_dev)
    x, lg = wide[:, 128:384], lgw[:, 3:11]
    want = moe.few_tokens_moe(x.contiguous(), lg.contiguous(), w13, s13, w2, s2, 2)
    big = torch.full((6, 300), 7.0, device=cuda_dev, dtype=torch.bfloat16)
    moe.few_tokens_moe(x, lg, w13, s13, w2, s2, 2, out=big[:, 5:261])
    assert torch.equal(big[:, 5:261], want) and (big[:, :5] == 7).all() and (big[:, 261:] == 7).all()
    y = x.contiguous()
    moe.few_tokens_moe(y, lg, w13, s13, w2, s2, 2, out=y)                # the first kernel has read x before the second writes
    assert torch.equal(y, want)


def test_repeatable_on_streams_and_in_graphs(cuda_dev):
    from kb_nano_b200 import moe, ops
    sets = [experts("fp8", 16, 1024, 512, cuda_dev, 13 + j) for j in range(2)]
    xs = [torch.randn(8, 1024, device=cuda_dev).to(torch.bfloat16) for _ in range(2)]
    lgs = [torch.randn(8, 16, device=cuda_dev) for _ in range(2)]

    def call(j, **kw):
        w13, s13, w2, s2, _, _ = sets[j]
        return moe.few_tokens_moe(xs[j], lgs[j], w13, s13, w2, s2, 4, **kw)

    want = [call(0), call(1)]
    assert torch.equal(call(0), want[0])                                 # sums in a fixed order
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(want[j]) for _ in range(4)] for j in range(2)]
    torch.cuda.synchronize()
    for r in range(4):
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                call(j, out=outs[j][r])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[j]) for j in range(2) for o in outs[j])
    graphs, gouts = [], []
    for j in range(2):
        o = torch.empty_like(want[j])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(j, out=o)
        graphs.append(g)
        gouts.append(o)
    torch.cuda.synchronize()
    for r in range(3):
        for o in gouts:
            o.zero_()
        torch.cuda.synchronize()
        for j in range(2):                                               # both graphs at once, each with memory of its own
            with torch.cuda.stream(streams[j]):
                graphs[j].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(gouts[j], want[j]) for j in range(2))
    assert ops.gemm_status(cuda_dev) == 0


def test_no_tokens(cuda_dev):
    from kb_nano_b200 import moe
    w13, s13, w2, s2, _, _ = experts("fp8", 2, 128, 128, cuda_dev, 14)
    out = moe.few_tokens_moe(torch.empty(0, 128, dtype=torch.bfloat16, device=cuda_dev), torch.empty(0, 2, device=cuda_dev), w13, s13, w2, s2, 1)
    assert tuple(out.shape) == (0, 128)


def test_refusals(cuda_dev):
    from kb_nano_b200 import moe
    from kb_nano_b200._lib import KbnError
    w13, s13, w2, s2, _, _ = experts("fp8", 4, 256, 128, cuda_dev, 15)
    x, lg = torch.zeros(2, 256, dtype=torch.bfloat16, device=cuda_dev), torch.zeros(2, 4, device=cuda_dev)
    with pytest.raises(ValueError, match="at most 16"):
        moe.few_tokens_moe(x[:1].expand(17, -1).contiguous(), lg[:1].expand(17, -1).contiguous(), w13, s13, w2, s2, 2)
    with pytest.raises(ValueError, match="bf16"):
        moe.few_tokens_moe(x.float(), lg, w13, s13, w2, s2, 2)
    with pytest.raises(ValueError, match="w13 must be"):
        moe.few_tokens_moe(x, lg, w13[:, :128].contiguous(), s13, w2, s2, 2)
    with pytest.raises(ValueError, match="w13_scale must be"):
        moe.few_tokens_moe(x, lg, w13, s13.to(torch.bfloat16), w2, s2, 2)
    with pytest.raises(ValueError, match="both"):
        moe.few_tokens_moe(x, lg, w13, s13, w2.view(torch.uint8), s2, 2)
    with pytest.raises(ValueError, match="come together"):
        moe.few_tokens_moe(x, lg, w13, s13, w2, s2, 2, out_ids=torch.empty(2, 2, dtype=torch.int32, device=cuda_dev))
    with pytest.raises(ValueError, match="CUDA tensors"):
        moe.few_tokens_moe(x, lg, w13.cpu(), s13, w2, s2, 2)
    for top in (5, 0, -1):
        with pytest.raises((KbnError, ValueError, RuntimeError)):
            moe.few_tokens_moe(x, lg, w13, s13, w2, s2, top)
    with pytest.raises(KbnError, match="16-byte"):
        off = torch.zeros(2, 264, dtype=torch.bfloat16, device=cuda_dev)[:, 1:257]
        moe.few_tokens_moe(off, lg, w13, s13, w2, s2, 2)


def test_layers_take_it_when_told_to(cuda_dev):
    """Qwen3MoE and DeepSeekMoE with use_few_tokens: both forms within their own error of the layer in 64 bits (the pipeline's is
    the FP8 rounding of its activations), larger batches and the default untouched, MixtralMoE refuses (its router weights
    are rounded to bf16)."""
    from types import SimpleNamespace

    from kb_nano_b200 import layers, moe, ops
    quant = {"weight_block_size": [128, 128]}
    e, h, i, top = 16, 512, 256, 4
    w13, s13, w2, s2, f13, f2 = experts("fp8", e, h, i, cuda_dev, 30)
    qwen = layers.Qwen3MoE(SimpleNamespace(num_experts=e, num_experts_per_tok=top, hidden_size=h, moe_intermediate_size=i, norm_topk_prob=True), quant)
    deep = layers.DeepSeekMoE(SimpleNamespace(n_routed_experts=e, num_experts_per_tok=top, hidden_size=h, moe_intermediate_size=i, n_group=4, topk_group=2,
                                              scoring_func="sigmoid", norm_topk_prob=True, topk_method="noaux_tc", n_shared_experts=None,
                                              routed_scaling_factor=1.5), quant)
    for layer, names in ((qwen, ("w13_scale", "w2_scale")), (deep, ("w13_weight_scale_inv", "w2_weight_scale_inv"))):
        layer.to(cuda_dev)
        layer.w13.data, layer.w2.data = w13, w2
        getattr(layer, names[0]).data, getattr(layer, names[1]).data = s13, s2
        gate = layer.gate.weight if layer is qwen else layer.gate_weight
        gate.data = (torch.randn(e, h, device=cuda_dev) * 0.1).to(torch.bfloat16)
        layer.requires_grad_(False)
        x = torch.randn(3, 4, h, device=cuda_dev).to(torch.bfloat16)
        before = layer(x)
        layer.use_few_tokens()
        got = layer(x)
        assert got.shape == x.shape and not torch.equal(got, before)
        flat, logits = x.view(12, h), torch.nn.functional.linear(x.view(12, h), gate)
        if layer is qwen:
            w, ids = ref.route(logits, top)
            factor = 1.0
        else:                                                     # bf16 scores and weights: taken from the routing kernel
            w, ids = ops.moe_route_topk(logits, top, "sigmoid", layer.e_score_correction_bias, 4, 2, True, round_bf16=True)
            factor = 1.5                                           # applied to the rounded bf16 result: one more rounding
        for out, fp8 in ((got, False), (before, True)):
            want, err = ref.moe(flat, f13, f2, w.double(), ids.long(), fp8)
            check(out.view(12, h), want * factor, err * factor + (want.abs() * factor * 2.0**-8 if factor != 1.0 else 0.0))
        big = torch.randn(20, h, device=cuda_dev).to(torch.bfloat16)
        many = layer(big)
        layer.use_few_tokens(0)
        assert torch.equal(layer(x), before) and torch.equal(layer(big), many)
        with pytest.raises(ValueError, match="at most"):
            layer.use_few_tokens(17)
    mixtral = layers.MixtralMoE(SimpleNamespace(num_local_experts=e, num_experts_per_tok=2, hidden_size=h, intermediate_size=i), quant)
    with pytest.raises(NotImplementedError):
        mixtral.use_few_tokens()
    assert ops.gemm_status(cuda_dev) == 0 and moe.FEW_TOKENS_MAX == 16


def test_registered_ops(cuda_dev):
    from kb_nano_b200 import moe, ops, torch_ops  # noqa: F401
    w13, s13, w2, s2, _, _ = experts("mxfp4", 4, 256, 128, cuda_dev, 31)
    x, lg = torch.randn(3, 256, device=cuda_dev).to(torch.bfloat16), torch.randn(3, 4, device=cuda_dev)
    out = torch.empty_like(x)
    torch.ops.kbn_b200.few_tokens_moe(x, lg, w13, s13, w2, s2, out, 2)
    assert torch.equal(out, moe.few_tokens_moe(x, lg, w13, s13, w2, s2, 2))
    q, s = torch.empty(3, 128, dtype=torch.uint8, device=cuda_dev), torch.empty(3, 8, dtype=torch.uint8, device=cuda_dev)
    torch.ops.kbn_b200.quant_mxfp4(x, q, s)
    assert torch.equal(q, ref.quant(x)[0]) and torch.equal(s, ref.quant(x)[1])
    wp, sf = ops.pack_mxfp4_scales(s2[0].contiguous(), 128), torch.empty(ops.packed_mxfp4_bytes(3, 128), dtype=torch.uint8, device=cuda_dev)
    y, y2 = torch.empty(3, 256, dtype=torch.bfloat16, device=cuda_dev), torch.empty(3, 256, dtype=torch.bfloat16, device=cuda_dev)
    half = x[:, :128].contiguous()
    torch.ops.kbn_b200.mxfp4_linear(half, q[:, :64].contiguous(), sf, w2[0], wp, y)
    ops.mxfp4_linear(half, q[:, :64].contiguous(), sf, w2[0], wp, y2)
    assert torch.equal(y, y2)


def test_two_gpus_worth_of_checks_on_one(cuda_dev):
    """Tensors that live on another device than the others are refused before anything is launched."""
    from kb_nano_b200 import moe
    w13, s13, w2, s2, _, _ = experts("fp8", 4, 256, 128, cuda_dev, 32)
    x, lg = torch.zeros(1, 256, dtype=torch.bfloat16, device=cuda_dev), torch.zeros(1, 4, device=cuda_dev)
    for bad in range(6):
        args = [x, lg, w13, s13, w2, s2]
        args[bad] = args[bad].cpu()
        with pytest.raises(ValueError, match="CUDA tensors|same device"):
            moe.few_tokens_moe(*args, 2)


def test_a_nan_logit_of_a_sigmoid_router_takes_one_expert_away(cuda_dev):
    """Seven of eight experts left for top-4, then three left: the fourth slot repeats the lowest choice, as ops.moe_route_topk does."""
    from kb_nano_b200 import moe, ops
    w13, s13, w2, s2, f13, f2 = experts("fp8", 8, 256, 128, cuda_dev, 33)
    x = torch.randn(3, 256, device=cuda_dev).to(torch.bfloat16)
    lg = torch.randn(3, 8, device=cuda_dev)
    lg[0, 2] = float("nan")
    lg[1, :5] = float("nan")
    ow, oi = torch.empty(3, 4, device=cuda_dev), torch.empty(3, 4, dtype=torch.int32, device=cuda_dev)
    got = moe.few_tokens_moe(x, lg, w13, s13, w2, s2, 4, "sigmoid", out_w=ow, out_ids=oi)
    w, ids = ops.moe_route_topk(lg, 4, "sigmoid")
    assert torch.equal(ow, w) and torch.equal(oi, ids.to(torch.int32))
    assert 2 not in oi[0].tolist() and min(oi[1].tolist()) >= 5
    want, err = ref.moe(x, f13, f2, w.double(), ids.long(), False)
    check(got, want, err)


def test_layers_refuse_what_the_kernels_do_not_take(cuda_dev):
    from types import SimpleNamespace

    from kb_nano_b200 import layers
    wide = layers.Qwen3MoE(SimpleNamespace(num_experts=32, num_experts_per_tok=17, hidden_size=256, moe_intermediate_size=128, norm_topk_prob=True),
                           {"weight_block_size": [128, 128]})
    with pytest.raises(ValueError, match="at most 16"):
        wide.use_few_tokens()
    wide.use_few_tokens(0)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,h,i,e,top", [(16, 256, 14336, 2, 1), (5, 128, 14336, 2, 2), (16, 128, 13696, 3, 2), (9, 256, 7296, 2, 2), (16, 128, 24576, 2, 1)])
def test_long_intermediate_rows_worked_on_in_parts(cuda_dev, fmt, t, h, i, e, top):
    """Rows too long for a full job's tokens beside the weights' ring: the second kernel takes K in two or four parts."""
    run_case(cuda_dev, fmt, t, h, i, e, top, seed=t + i)


def test_native_call_accepts_what_the_checks_accept(cuda_dev):
    """The native call path takes a well-formed call of either format (every optional argument given or not) and answers False to one
    wrong argument at a time, whatever it is; the public function then raises, or does what it did before for an odd type."""
    from kb_nano_b200 import _lib, moe, ops
    native = _lib.calls().few_tokens_moe
    for fmt in ("fp8", "mxfp4"):
        w13, s13, w2, s2, _, _ = experts(fmt, 8, 256, 128, cuda_dev, 34)
        x, lg, bias = torch.randn(3, 256, device=cuda_dev).to(torch.bfloat16), torch.randn(3, 8, device=cuda_dev), torch.randn(8, device=cuda_dev) * 0.1
        out, ow, oi = torch.empty_like(x), torch.empty(3, 2, device=cuda_dev), torch.empty(3, 2, dtype=torch.int32, device=cuda_dev)
        full = (x, lg, w13, s13, w2, s2, 2, "sigmoid", bias, 2, 1, True, 0.0, 1.0, False, out, ow, oi)
        plain = (x, lg.to(torch.bfloat16), w13, s13, w2, s2, 2, "softmax", None, 1, 1, False, 0.0, 2.5, True, None, None, None)
        assert native(*full) is out
        fresh = native(*plain)
        assert fresh.shape == x.shape and fresh.dtype == x.dtype and fresh.is_contiguous()
        assert torch.equal(fresh, moe.few_tokens_moe(*plain))
        for i, a in enumerate(full):
            if isinstance(a, torch.Tensor):
                bads = [a.cpu(), a.double(), a[:0], a[..., :-1], 3, None if i in (0, 1, 2, 3, 4, 5) else "x"]
            else:
                bads = {6: [0, 9, 17, "2", None], 7: ["tanh", 1, None], 9: [3, 0, None], 10: [3, 0, None], 11: [None], 12: [None], 13: [None], 14: [None]}[i]
            for bad in bads:
                args = (*full[:i], bad, *full[i + 1:])
                assert native(*args) is False, (fmt, i, bad)
                if isinstance(bad, torch.Tensor) and bad.numel() or i in (6, 7, 9, 10) and isinstance(bad, int):
                    with pytest.raises((ValueError, RuntimeError, TypeError)):
                        moe.few_tokens_moe(*args)
        assert torch.equal(moe.few_tokens_moe(*full[:13], 1, *full[14:]), native(*full))      # an int factor: through the checks
        assert native() is False and native(*full[:-1]) is False
    assert ops.gemm_status(cuda_dev) == 0


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,i", [(1, 65536), (3, 102400), (16, 32896)])
def test_intermediate_rows_longer_than_shared_memory(cuda_dev, fmt, t, i):
    run_case(cuda_dev, fmt, t, 128, i, 1, 1, seed=t + i)
