"""The C-ABI kernels as opaque torch.library custom ops (namespace ``kbn_b200``).

kb-nano wraps its FP8 kernels the same way (``torch.ops.kb_nano_fp8.*``,
tasks/baseline/L1/fp8_linear.py:85-178; ``torch.ops.kb_nano_fp8_moe.*``,
tasks/baseline/L1/fp8_grouped_gemm_contiguous.py:100-133) so that torch.compile treats them as
single in-place nodes and never traces into them.  Outputs are caller-allocated and mutated.
"""
from __future__ import annotations

import torch

from . import moe, ops


@torch.library.custom_op("kbn_b200::per_token_group_quant_fp8", mutates_args=("output_fp8", "output_scale"))
def per_token_group_quant_fp8(input: torch.Tensor, output_fp8: torch.Tensor, output_scale: torch.Tensor,
                              use_ue8m0: bool = True, eps: float = 1e-10) -> None:
    ops.per_token_group_quant_fp8(input, output_fp8, output_scale, use_ue8m0, eps)


@torch.library.custom_op("kbn_b200::silu_mul_quant_fp8", mutates_args=("output_fp8", "output_scale"))
def silu_mul_quant_fp8(input: torch.Tensor, output_fp8: torch.Tensor, output_scale: torch.Tensor,
                       use_ue8m0: bool = True, eps: float = 1e-10) -> None:
    ops.silu_mul_quant_fp8(input, output_fp8, output_scale, use_ue8m0, eps)


@torch.library.custom_op("kbn_b200::fp8_gemm_nt", mutates_args=("output",))
def fp8_gemm_nt(a_fp8: torch.Tensor, a_scale: torch.Tensor, b_fp8: torch.Tensor, b_scale: torch.Tensor,
                output: torch.Tensor) -> None:
    ops.fp8_gemm_nt_auto(a_fp8, a_scale, b_fp8, b_scale, output)


@torch.library.custom_op("kbn_b200::m_grouped_gemm_nt_contiguous", mutates_args=("c_bf16",))
def m_grouped_gemm_nt_contiguous(a_fp8: torch.Tensor, a_scale: torch.Tensor, b_fp8: torch.Tensor,
                                 b_scale: torch.Tensor, c_bf16: torch.Tensor, expert_ids: torch.Tensor) -> None:
    ops.m_grouped_fp8_gemm_nt_contiguous(a_fp8, a_scale, b_fp8, b_scale, c_bf16, expert_ids)


@torch.library.custom_op("kbn_b200::m_grouped_gemm_nt_masked", mutates_args=("c_bf16",))
def m_grouped_gemm_nt_masked(a_fp8: torch.Tensor, a_scale: torch.Tensor, b_fp8: torch.Tensor,
                             b_scale: torch.Tensor, c_bf16: torch.Tensor, masked_m: torch.Tensor) -> None:
    ops.m_grouped_fp8_gemm_nt_masked(a_fp8, a_scale, b_fp8, b_scale, c_bf16, masked_m)


# The 4-bit counterparts and the MoE layer for a few tokens (no counterpart in kb-nano).

@torch.library.custom_op("kbn_b200::quant_mxfp4", mutates_args=("output_fp4", "output_scale"))
def quant_mxfp4(input: torch.Tensor, output_fp4: torch.Tensor, output_scale: torch.Tensor) -> None:
    ops.quant_mxfp4(input, output_fp4, output_scale)


@torch.library.custom_op("kbn_b200::silu_mul_quant_mxfp4", mutates_args=("output_fp4", "output_scale"))
def silu_mul_quant_mxfp4(input: torch.Tensor, output_fp4: torch.Tensor, output_scale: torch.Tensor) -> None:
    ops.silu_mul_quant_mxfp4(input, output_fp4, output_scale)


@torch.library.custom_op("kbn_b200::mxfp4_linear", mutates_args=("a_fp4", "a_packed", "output"))
def mxfp4_linear(input: torch.Tensor, a_fp4: torch.Tensor, a_packed: torch.Tensor, b_fp4: torch.Tensor, b_packed: torch.Tensor,
                 output: torch.Tensor, bias: torch.Tensor | None = None) -> None:
    ops.mxfp4_linear(input, a_fp4, a_packed, b_fp4, b_packed, output, bias)


@torch.library.custom_op("kbn_b200::few_tokens_moe", mutates_args=("output",))
def few_tokens_moe(hidden_states: torch.Tensor, router_logits: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor,
                   w2_scale: torch.Tensor, output: torch.Tensor, top_k: int, scoring: str = "softmax", bias: torch.Tensor | None = None,
                   n_group: int = 1, topk_group: int = 1, renormalize: bool = True, renorm_floor: float = 0.0, scale: float = 1.0, round_bf16: bool = False) -> None:
    moe.few_tokens_moe(hidden_states, router_logits, w13, w13_scale, w2, w2_scale, top_k, scoring, bias, n_group, topk_group, renormalize,
                       renorm_floor, scale, round_bf16, out=output)
