"""The few-token MoE layer where other code reaches it: the registered op, the layer classes."""
import pytest
import torch

from tests.test_moe_few_gpu import experts

pytestmark = pytest.mark.gpu


def test_registered_op_rounds_scores_as_deepseek_does(cuda_dev):
    """bf16 logits scored and weighed in bf16 steps: the registered op gives what the function gives, and other than without."""
    from kb_nano_b200 import moe, ops, torch_ops  # noqa: F401
    e, h, i, top = 16, 512, 256, 4
    w13, s13, w2, s2, _, _ = experts("fp8", e, h, i, cuda_dev, 50)
    x, bias = torch.randn(7, h, device=cuda_dev).to(torch.bfloat16), torch.randn(e, device=cuda_dev) * 0.1
    lg = torch.randn(7, e, device=cuda_dev).to(torch.bfloat16)
    outs = [torch.empty_like(x) for _ in range(2)]
    for rounds in (False, True):
        torch.ops.kbn_b200.few_tokens_moe(x, lg, w13, s13, w2, s2, outs[rounds], top, "sigmoid", bias, 4, 2, True, 0.0, 1.0, rounds)
        assert torch.equal(outs[rounds], moe.few_tokens_moe(x, lg, w13, s13, w2, s2, top, "sigmoid", bias, 4, 2, round_bf16=rounds))
    assert not torch.equal(outs[0], outs[1])
    by_default = torch.empty_like(x)
    torch.ops.kbn_b200.few_tokens_moe(x, lg, w13, s13, w2, s2, by_default, top, "sigmoid", bias, 4, 2)
    assert torch.equal(by_default, outs[0]) and ops.gemm_status(cuda_dev) == 0


def test_layers_take_tokens_from_any_address(cuda_dev):
    """Contiguous tokens that do not start on a 16-byte boundary: taken by a layer with use_few_tokens as by one without."""
    from types import SimpleNamespace

    from kb_nano_b200 import layers, ops
    e, h, i, top = 8, 256, 128, 2
    w13, s13, w2, s2, _, _ = experts("fp8", e, h, i, cuda_dev, 51)
    layer = layers.Qwen3MoE(SimpleNamespace(num_experts=e, num_experts_per_tok=top, hidden_size=h, moe_intermediate_size=i, norm_topk_prob=True),
                            {"weight_block_size": [128, 128]}).to(cuda_dev)
    layer.w13.data, layer.w2.data, layer.w13_scale.data, layer.w2_scale.data = w13, w2, s13, s2
    layer.gate.weight.data = (torch.randn(e, h, device=cuda_dev) * 0.1).to(torch.bfloat16)
    layer.requires_grad_(False)
    buf = torch.randn(5 * h + 1, device=cuda_dev).to(torch.bfloat16)
    x = buf[1:].view(5, h)
    for few in (0, 16):
        layer.use_few_tokens(few)
        assert torch.equal(layer(x), layer(x.clone()))
    assert ops.gemm_status(cuda_dev) == 0
