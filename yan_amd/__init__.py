"""MI355X-native GEMM hot path behind the JIT / operator surface of zoheth/yan (`yan/__init__.py:3-5`)."""
import torch

from . import jit
from .jit_kernels import (gemm, gemm_float_nt, gemm_bf16_tn, gemm_fp16_tn, gemm_bf16_fp8_bf16_nt, gemm_fp8_fp8_bf16_nt, get_col_major_tensor,
                          m_grouped_gemm_fp8_fp8_bf16_nt_contiguous, m_grouped_gemm_fp8_fp8_bf16_nt_masked,
                          per_token_cast_to_fp8, per_block_cast_to_fp8, per_channel_cast_to_fp8,
                          gemm_fp8_fp8_fp32_nt, k_grouped_gemm_fp8_fp8_fp32_nt_contiguous,
                          moe_route, moe_route_backward, moe_dispatch_to_fp8_contiguous, moe_dispatch_to_fp8_masked, moe_combine, moe_combine_backward,
                          get_contiguous_layout_rows, moe_ragged_layout,
                          m_grouped_gemm_bf16_bf16_bf16_nt_ragged, m_grouped_gemm_fp16_fp16_fp16_nt_ragged, m_grouped_gemm_bf16_bf16_bf16_nn_ragged,
                          m_grouped_gemm_fp16_fp16_fp16_nn_ragged, k_grouped_gemm_bf16_bf16_fp32_tn_ragged, k_grouped_gemm_fp16_fp16_fp32_tn_ragged,
                          rms_norm, rms_norm_to_fp8, rms_norm_backward,
                          set_num_sms, get_num_sms, ceil_div, get_m_alignment_for_contiguous_layout)
from .utils import bench_kineto, calc_diff, count_bytes
