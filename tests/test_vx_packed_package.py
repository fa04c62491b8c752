"""The Vx declarations and wrappers of the packed batch's ops
(vx_amd/vx/packages/vx_nn/lib.vx) against the C header, as test_vx_package.py holds
the others'."""

import pytest

from tests import test_vx_package as vx

OPS = ["vx_nn_rms_norm_bf16", "vx_nn_rms_norm_f32", "vx_nn_quantize_i8_bf16", "vx_nn_quantize_i8_f32",
       "vx_nn_gemm_i8_bf16", "vx_nn_gemm_i8_f32", "vx_nn_gemm_i8_workspace", "vx_nn_flash_attention_packed_bf16",
       "vx_nn_token_logprobs_f32", "vx_nn_token_logprobs_bf16", "vx_nn_token_logprobs_workspace"]


@pytest.mark.parametrize("op", OPS)
def test_declared_as_in_the_header(op):
    vx.test_declared_as_in_the_header(op)


def test_no_op_is_left_out():
    """Every op the header declares is compared here or there."""
    assert {n for n in vx.in_c() if n.startswith("vx_nn_")} <= set(OPS) | set(vx.OPS)


@pytest.mark.parametrize("name", ["rms_norm_i8", "quantize_i8", "gemm_i8", "flash_attention_packed", "token_logprobs"])
def test_wrappers_pass_what_the_op_takes(name):
    vx.test_wrappers_pass_what_the_op_takes(name)
