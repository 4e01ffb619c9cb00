"""What the MXFP4 and few-token entry points refuse before any GPU work: argument checks of the C ABI with made-up addresses
(nothing is dereferenced) and of the tensor-level calls with CPU tensors.  The 64-bit restatements the GPU tests compare with
are checked here against values worked out by hand."""
import pytest
import torch

from tests import mx_reference as ref

A = 1 << 20          # an aligned, never dereferenced address


def refused(lib, rc, word):
    assert rc < 0 and word.encode() in lib.kbn_last_error(), (rc, lib.kbn_last_error())


def test_quant_arguments(kbn_lib):
    q = kbn_lib.kbn_quant_mxfp4
    refused(kbn_lib, q(A, 4, 48, 48, A, 24, A, 1, None, None), "multiple of 32")
    refused(kbn_lib, q(None, 4, 64, 64, A, 32, A, 2, None, None), "null")
    refused(kbn_lib, q(A, 4, 64, 32, A, 32, A, 2, None, None), "row stride")
    refused(kbn_lib, q(A, 4, 64, 64, A, 33, A, 2, None, None), "4-byte")
    refused(kbn_lib, q(A, 4, 64, 64, A, 32, A, 1, None, None), "scale row stride")
    refused(kbn_lib, q(A, 4, 64, 64, A, 32, None, 0, None, None), "no place for the scales")
    refused(kbn_lib, q(A, 4, 64, 64, A, 32, None, 0, A + 4, None), "16-byte")
    refused(kbn_lib, q(A, -1, 64, 64, A, 32, A, 2, None, None), "negative")
    assert q(None, 0, 64, 64, None, 32, None, 2, None, None) == 0
    refused(kbn_lib, kbn_lib.kbn_silu_mul_quant_mxfp4(A, 4, 64, 64, A, 32, A, 2, None, None), "row stride")
    refused(kbn_lib, kbn_lib.kbn_dequant_mxfp4(A, 32, A, 2, 4, 64, A + 1, 64, None), "odd")
    refused(kbn_lib, kbn_lib.kbn_pack_mxfp4_scales(A, 4, 64, 2, A + 8, None), "16-byte")
    assert kbn_lib.kbn_packed_mxfp4_bytes(129, 160) == 2 * 2 * 512


def test_gemm_arguments(kbn_lib):
    g, lin = kbn_lib.kbn_mxfp4_gemm_nt, kbn_lib.kbn_mxfp4_linear
    refused(kbn_lib, g(A, A, A, A, None, A, 16, 4, 16, 40, None), "multiple of 32")
    refused(kbn_lib, g(A + 8, A, A, A, None, A, 16, 4, 16, 64, None), "16-byte")
    refused(kbn_lib, g(A, A, A, A, None, A, 8, 4, 16, 64, None), "row stride")
    refused(kbn_lib, g(A, None, A, A, None, A, 16, 4, 16, 64, None), "null")
    refused(kbn_lib, g(A, A, A, A, None, A, 16, 1 << 30, 16, 64, None), "too large")
    assert g(None, None, None, None, None, None, 16, 0, 16, 64, None) == 0
    refused(kbn_lib, lin(A, 32, 4, 64, A, A, A, A, None, A, 16, 16, None), "stride")
    refused(kbn_lib, lin(A, 64, 4, 64, None, A, A, A, None, A, 16, 16, None), "null")
    assert lin(A, 64, 4, 64, A, A, A, A, None, A, 16, 0, None) == 0


def test_linear_refuses_an_output_on_top_of_its_input(kbn_lib):
    lin = kbn_lib.kbn_mxfp4_linear
    for ld_x, m, c, ldc in [(64, 4, A, 64), (64, 4, A + 32, 64), (64, 1, A + 126, 16), (64, 1, A - 30, 16), (256, 4, A + 3 * 512 + 96, 16), (256, 4, A + 512 - 16, 256)]:
        refused(kbn_lib, lin(A, ld_x, m, 64, 2 * A, 2 * A, 2 * A, 2 * A, None, c, ldc, 16, None), "overlap")


def moe_args(**kw):
    d = dict(x=A, ld_x=256, T=2, logits=A, bf16=0, ld=8, E=8, softmax=1, bias=None, n_group=1, topk_group=1, topk=2, renorm=1, floor=0.0, scale=1.0, round=0,
             fmt=0, w13=A, s13=A, w2=A, s2=A, H=256, I=128, out=A, ld_out=256, ow=None, oi=None, ws=A, wb=1 << 30)
    d.update(kw)
    return (*d.values(), None)


@pytest.mark.parametrize("change,word", [(dict(T=17), "at most 16 tokens"), (dict(E=2000, ld=2000), "at most 1024"), (dict(topk=17, E=64, ld=64), "topk"), (dict(topk=9), "topk"),
                                         (dict(H=200), "multiples of 128"), (dict(I=64), "multiples of 128"), (dict(fmt=2), "weight_format"),
                                         (dict(n_group=3), "n_group"), (dict(n_group=4, topk_group=1, topk=3), "fewer experts"), (dict(x=None), "null"),
                                         (dict(ow=A), "come together"), (dict(ld_x=128), "stride"), (dict(x=A + 2), "16-byte"), (dict(w2=A + 8), "16-byte"),
                                         (dict(wb=100), "workspace"), (dict(T=-1), "bad sizes"), (dict(E=1024, ld=1024, H=128, I=1 << 21), "2^31")])
def test_moe_arguments(kbn_lib, change, word):
    refused(kbn_lib, kbn_lib.kbn_moe_few_tokens(*moe_args(**change)), word)


def test_moe_without_tokens_is_a_no_op(kbn_lib):
    assert kbn_lib.kbn_moe_few_tokens(*moe_args(T=0, x=None, logits=None, out=None, ws=None, wb=0)) == 0
    assert kbn_lib.kbn_moe_few_tokens_workspace_bytes(0, 2, 256, 128) == 0
    small, large = (kbn_lib.kbn_moe_few_tokens_workspace_bytes(t, 8, 7168, 2048) for t in (1, 16))
    assert 8 * (7168 + 2048) * 4 <= small < large and large < 8 << 20


def test_tensor_calls_refuse_cpu_tensors(kbn_lib):
    from kb_nano_b200 import moe, ops
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    q, s, p = torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), torch.zeros(1 << 12, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.quant_mxfp4(x, q, s)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.silu_mul_quant_mxfp4(torch.zeros(2, 256, dtype=torch.bfloat16), q, s)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.dequant_mxfp4(q, s, x)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.pack_mxfp4_scales(s, 128)
    with pytest.raises(ValueError, match="CUDA tensors|16-byte"):
        ops.mxfp4_linear(x, q, p, q, p, torch.zeros(2, 2, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA tensors"):
        moe.few_tokens_moe(x, torch.zeros(2, 4), torch.zeros(4, 256, 128, dtype=torch.float8_e4m3fn), torch.ones(4, 2, 1), torch.zeros(4, 128, 128, dtype=torch.float8_e4m3fn),
                           torch.ones(4, 1, 1), 2)


def test_reference_quantiser_by_hand():
    x = torch.zeros(1, 64)
    x[0, :6] = torch.tensor([6.0, 0.25, 0.75, 2.5, -5.0, 3.5])      # scale 2^0; midpoints to even codes
    x[0, 32] = 6.5                                                    # does not fit 6 * 2^0: scale 2^1, 3.25 -> 3
    q, s = ref.quant(x)
    assert s.tolist() == [[127, 128]]
    assert ref.values(q, s)[0, :6].tolist() == [6.0, 0.0, 1.0, 2.0, -4.0, 4.0]
    assert ref.values(q, s)[0, 32].item() == 6.0
    x[0, 1] = float("inf")
    q, s = ref.quant(x)
    assert s.tolist() == [[255, 128]] and torch.isnan(ref.values(q, s)[0, :32]).all()
    assert ref.pack_scales(s).numel() == 512 and ref.pack_scales(s)[:4].tolist() == [255, 128, 127, 127]


def test_reference_routing_by_hand():
    w, ids = ref.route(torch.tensor([[0.0, 0.0, 1.0, 0.0]]), 3)
    assert ids.tolist() == [[2, 0, 1]] and abs(w.sum().item() - 1) < 1e-12
    w, ids = ref.route(torch.tensor([[5.0, -9.0, 1.0, 1.5]]), 1, "sigmoid", torch.zeros(4), n_group=2, topk_group=1)
    assert ids.tolist() == [[3]]                                      # 1 + 2 of group two beat 5 and -9: sums of the two best


def test_native_calls_accept_nothing_that_is_not_a_cuda_tensor(kbn_lib):
    """The native call path answers False, without an exception, for what it does not know; the Python checks then say why."""
    from kb_nano_b200 import _lib
    calls = _lib.calls()
    x, q, s, p = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), torch.zeros(1 << 12, dtype=torch.uint8)
    out = torch.zeros(2, 2, dtype=torch.bfloat16)
    for fn, args in ((calls.quant_mxfp4, (x, q, s, None)), (calls.silu_mul_quant_mxfp4, (torch.zeros(2, 256, dtype=torch.bfloat16), q, s, p)),
                     (calls.dequant_mxfp4, (q, s, x)), (calls.mxfp4_gemm_nt, (q, p, q, p, out, None)), (calls.mxfp4_linear, (x, q, p, q, p, out, None))):
        assert fn(*args) is False
        for i in range(len(args)):
            for bad in (None, 3, "x", object(), torch.Tensor, torch.zeros(2, 128, device="meta"), torch.zeros(()), torch.eye(2).to_sparse()):
                assert fn(*args[:i], bad, *args[i + 1:]) is False
        assert fn() is False and fn(*args, None) is False and fn(*args[:-1]) is False


def test_moe_refuses_token_rows_longer_than_shared_memory(kbn_lib):
    for fmt in (0, 1):
        refused(kbn_lib, kbn_lib.kbn_moe_few_tokens(*moe_args(H=131072, ld_x=131072, ld_out=131072, fmt=fmt, wb=1 << 40)), "shared memory")
