"""Pointers that are not aligned to their elements are refused by the C entry points before any GPU work (made-up addresses,
nothing is dereferenced)."""
import pytest

from tests.test_mxfp4_cpu import A, moe_args, refused


@pytest.mark.parametrize("change", [dict(logits=A + 2), dict(logits=A + 1, bf16=1), dict(bias=A + 2), dict(out=A + 1), dict(ow=A + 2, oi=A), dict(ow=A, oi=A + 1)])
def test_moe(kbn_lib, change):
    refused(kbn_lib, kbn_lib.kbn_moe_few_tokens(*moe_args(**change)), "aligned to their elements")


@pytest.mark.parametrize("m", [4, 40])
def test_bias_of_gemm_and_linear(kbn_lib, m):
    refused(kbn_lib, kbn_lib.kbn_mxfp4_gemm_nt(A, A, A, A, A + 1, A, 16, m, 16, 128, None), "odd bias")
    refused(kbn_lib, kbn_lib.kbn_mxfp4_linear(A, 128, m, 128, 2 * A, 2 * A, 2 * A, 2 * A, 2 * A + 1, 3 * A, 16, 16, None), "odd bias")
