"""FP8 products of weight gradients: both operands quantised 1 x 128 along K with power-of-two scales, fp32 sums into fp32 gradients.

The reference's FP8 template has one scale per row and K block on one side and per 128 x 128 block on the other (`yan/jit_kernels/gemm.py:8-31`,
`yan/include/gemm/fp8_gemm.cuh:55-61`), which is what a forward pass and the gradient of activations need. A weight gradient contracts over
the tokens, so both of its operands have their scales along K; `per_channel_cast_to_fp8` makes them.

    out[i, j] (+)= sum_b 2^(lhs_scales[i, b] - 127) * 2^(rhs_scales[j, b] - 127) * sum_{t < 128} f32(lhs[i, 128 b + t]) * f32(rhs[j, 128 b + t])
"""
import functools
from typing import Optional, Tuple

import torch

from .host_calls import WGRAD, remember_new, repeat_call
from .tuner import FrozenKeys, jit_tuner
from .split_k import SPLIT_K_WORKSPACE_BYTES, split_k_launch_failed, split_k_workspace
from .utils import assert_on_current_device, ceil_div, current_raw_stream, get_num_sms

includes = ('"gemm/fp8_wgrad.hpp"', )

template = """
using namespace yan;
// Templated args from Python JIT call: {KERNEL} (kWgradAny: what wgrad_plan says) in {PARTS} parts
__return_code = static_cast<int>(launch_fp8_wgrad<{KERNEL}, {PARTS}>(lhs, lhs_scales, ld_lhs_scales, rhs, rhs_scales, ld_rhs_scales, out, grouped ? offsets : nullptr,
                                                                    groups, m, n, k, accumulate != 0, workspace_bytes ? workspace : nullptr, num_sms, stream));
"""

arg_defs = (('lhs', torch.float8_e4m3fn), ('lhs_scales', torch.uint8), ('rhs', torch.float8_e4m3fn), ('rhs_scales', torch.uint8), ('out', torch.float),
            ('offsets', torch.int), ('workspace', torch.uint8), ('ld_lhs_scales', int), ('ld_rhs_scales', int), ('grouped', int), ('groups', int), ('m', int), ('n', int), ('k', int),
            ('accumulate', int), ('workspace_bytes', int), ('num_sms', int), ('stream', torch.cuda.Stream))

MAX_K, MAX_N = 1 << 23, 1 << 21


@functools.lru_cache(maxsize=None)
def wgrad_kernel_plan(kernel: str = 'kWgradAny', parts: int = 1):
    """(name, keys, arg_defs, template) of the weight-gradient kernels; needs no GPU. The entries let `wgrad_plan` of gemm/fp8_wgrad.hpp choose."""
    return 'fp8_wgrad', FrozenKeys({'KERNEL': kernel, 'PARTS': parts}), arg_defs, template


def _check_operand(codes, scales):
    assert codes.dim() == 2 and codes.dtype == torch.float8_e4m3fn and codes.is_contiguous()
    rows, k = codes.shape
    assert k % 128 == 0 and k < MAX_K
    assert scales.shape == (rows, k // 128) and scales.dtype == torch.uint8
    assert scales.size(1) <= 1 or scales.stride(1) == 1
    if rows and k:
        assert scales.stride(0) % 4 == 0 and ceil_div(k, 512) * 4 <= scales.stride(0) < MAX_K and scales.data_ptr() % 4 == 0, \
            'rows of scales are whole groups of four bytes, as per_channel_cast_to_fp8 lays them out'
        assert codes.data_ptr() % 16 == 0


def _wgrad(lhs, rhs, out, offsets: Optional[torch.Tensor], accumulate: bool, kernel: tuple = ()) -> None:
    (lhs, lhs_scales), (rhs, rhs_scales) = lhs, rhs
    call = (WGRAD, lhs, lhs_scales, rhs, rhs_scales, out, offsets, 1 if accumulate else 0)
    if kernel == () and repeat_call(*call):
        return
    _check_operand(lhs, lhs_scales)
    _check_operand(rhs, rhs_scales)
    m, n, k = lhs.size(0), rhs.size(0), lhs.size(1)
    assert rhs.size(1) == k and n % 4 == 0 and n < MAX_N and out.shape[-2:] == (m, n)
    assert out.dtype == torch.float32 and out.is_contiguous() and out.data_ptr() % 16 == 0
    assert_on_current_device(lhs, lhs_scales, rhs, rhs_scales, out, offsets)
    if out.numel() == 0:
        return
    if k == 0:
        if not accumulate:
            out.zero_()
        return
    stream = current_raw_stream()
    workspace, token = split_k_workspace(out.device, stream)
    nothing = torch.empty(1, dtype=torch.int32, device=out.device)          # stands for what is not there
    args = (lhs, lhs_scales, rhs, rhs_scales, out, nothing if offsets is None else offsets, nothing.view(torch.uint8) if workspace is None else workspace,
            lhs_scales.stride(0), rhs_scales.stride(0), int(offsets is not None), 1 if offsets is None else out.size(0), m, n, k, int(bool(accumulate)),
            0 if workspace is None else SPLIT_K_WORKSPACE_BYTES, get_num_sms(), stream)
    name, keys, defs, code_template = wgrad_kernel_plan(*kernel)
    runtime = jit_tuner.compile_and_tune(name=name, keys=keys, space=(), includes=includes, arg_defs=defs, template=code_template, args=args)
    rc = runtime(*args)
    if rc != 0 and token is not None:
        split_k_launch_failed(token)
    assert rc == 0, f'{name} failed with HIP error {rc}'
    if kernel == ():
        remember_new(call, name, runtime, args, workspace=workspace)


def gemm_fp8_fp8_fp32_nt(lhs: Tuple[torch.Tensor, torch.Tensor], rhs: Tuple[torch.Tensor, torch.Tensor], out: torch.Tensor, accumulate: bool = False) -> None:
    """
    `out = lhs @ rhs.T`, or `out += lhs @ rhs.T`, of the decoded operands.

    lhs: (e4m3fn `[m, k]`, uint8 `[m, k/128]`), rhs: (e4m3fn `[n, k]`, uint8 `[n, k/128]`): codes contiguous; scales are exponents + 127 (E8M0), their
         rows contiguous and a multiple of 4 bytes apart, as `per_channel_cast_to_fp8` returns both. Bytes of 10 to 246 are exact for every code: a code
         times its scale is multiplied as bf16, and beyond them it may leave bf16's normal numbers (the cast's stay inside for values up to 3.2e38).
    out: fp32 `[m, n]` contiguous, written in place
    Requires k % 128 == 0 and n % 4 == 0; m is arbitrary.
    """
    assert out.dim() == 2
    _wgrad(lhs, rhs, out, None, accumulate)


def k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(lhs: Tuple[torch.Tensor, torch.Tensor], rhs: Tuple[torch.Tensor, torch.Tensor], out: torch.Tensor,
                                              offsets: torch.Tensor, accumulate: bool = False) -> None:
    """
    The weight gradients of all experts: K is cut into groups, and `out[g]` is the product over the columns of group g.

    lhs, rhs: as for `gemm_fp8_fp8_fp32_nt`, k the total number of rows of the contiguous layout (a row that no token has: zero codes)
    out: fp32 `[num_groups, m, n]` contiguous, written in place; a group without columns is zero, or unchanged with `accumulate`
    offsets: int32 `[num_groups + 1]`, ascending multiples of 128: group g has the columns offsets[g] .. offsets[g + 1] - 1, as
             `moe_dispatch_to_fp8_contiguous` returns them
    """
    assert out.dim() == 3 and out.size(0) > 0
    assert offsets.shape == (out.size(0) + 1, ) and offsets.dtype == torch.int32 and offsets.is_contiguous()
    _wgrad(lhs, rhs, out, offsets, accumulate)
