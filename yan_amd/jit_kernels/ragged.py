"""Products of 16-bit experts on groups of any number of rows, which `offsets` on the device cut out of one tensor: forward, for the gradient of the rows and for
the gradient of the weights.

The reference's grouped hooks (`yan/include/gemm/scheduler.cuh:7-11,31-48`) pad every group to a multiple of 128 rows, for FP8 (`yan/jit_kernels/utils.py:46-55`). A layer that
stays in 16 bits needs neither: its rows follow each other as `moe_ragged_layout` numbers them, and are gathered out of the tokens by the product itself.

    rows, source, offsets = moe_ragged_layout(indices, num_experts)
    m_grouped_gemm_bf16_bf16_bf16_nt_ragged(x, w1, y1, offsets, source)             # y1[r] = x[source[r]] @ w1[g].T
    m_grouped_gemm_bf16_bf16_bf16_nt_ragged(h, w2, y2, offsets)                     # h = act(y1)
    moe_combine(y2, rows, weights, out)

and back: `moe_combine_backward` for the gradients of y2, then of every product the two of

    m_grouped_gemm_bf16_bf16_bf16_nn_ragged(grad_y2, w2, grad_h, offsets)           # grad_h[r] = grad_y2[r] @ w2[g]
    k_grouped_gemm_bf16_bf16_fp32_tn_ragged(grad_y2, h, grad_w2, offsets, True)     # grad_w2[g] += grad_y2[rows of g].T @ h[rows of g]

and `moe_combine` without weights for the gradient of the tokens. Groups come with the padding of `moe_dispatch_to_fp8_contiguous` as well.
"""
import functools
from typing import Optional

import torch

from .host_calls import RAGGED_NN, RAGGED_NT, RAGGED_TN, remember_new, repeat_call
from .tuner import FrozenKeys, jit_tuner
from .utils import assert_on_current_device, current_raw_stream, get_num_sms

includes = ('"gemm/grouped16.hpp"', )

template = """
using namespace yan;
// Templated args from Python JIT call: elements {ELEMENT}, product {MODE}, gathered rows {GATHER}, {KERNEL} (kGroupedAny: what grouped16_plan says)
__return_code = static_cast<int>(launch_grouped16<{ELEMENT}, Grouped::{MODE}, {GATHER}, {KERNEL}>(
    lhs, rhs, out, offsets, {GATHER} ? source : nullptr, groups, rows, m, n, k, source_rows, accumulate != 0, num_sms, stream));
"""

# kGroupedMostRows and kGroupedMostColumns of gemm/grouped16.hpp; what a gathered operand may hold
MAX_ROWS, MAX_COLUMNS, MAX_GATHERED_BYTES = 1 << 29, 1 << 21, 1 << 31
MAX_GROUPS = 1024
_ELEMENTS = {torch.bfloat16: '__bf16', torch.half: '_Float16'}


def _arg_defs(dtype, out):
    return (('lhs', dtype), ('rhs', dtype), ('out', out), ('offsets', torch.int), ('source', torch.int), ('groups', int), ('rows', int), ('m', int), ('n', int), ('k', int),
            ('source_rows', int), ('accumulate', int), ('num_sms', int), ('stream', torch.cuda.Stream))


@functools.lru_cache(maxsize=None)
def grouped16_kernel_plan(dtype: torch.dtype, mode: str, gather: bool, kernel: str = 'kGroupedAny'):
    """(name, keys, arg_defs, template) of a ragged product's kernels; needs no GPU. The entries let `grouped16_plan` of gemm/grouped16.hpp choose."""
    keys = FrozenKeys({'ELEMENT': _ELEMENTS[dtype], 'MODE': mode, 'GATHER': 'true' if gather else 'false', 'KERNEL': kernel})
    return 'grouped16', keys, _arg_defs(dtype, torch.float32 if mode == 'TN' else dtype), template


def _check(dtype, lhs, rhs, out, offsets, groups, source):
    assert lhs.dtype == dtype and rhs.dtype == dtype and lhs.is_contiguous() and rhs.is_contiguous() and out.is_contiguous()
    assert offsets.shape == (groups + 1, ) and offsets.dtype == torch.int32 and offsets.is_contiguous()
    assert 0 < groups <= MAX_GROUPS and lhs.size(0) < MAX_ROWS
    for t in (lhs, rhs, out):
        assert t.data_ptr() % 16 == 0, 'tensors start at multiples of 16 bytes'
    if source is not None:
        assert source.dim() == 1 and source.dtype == torch.int32 and source.is_contiguous()


def _launch(call, dtype, mode, lhs, rhs, out, offsets, source, groups, rows, m, n, k, source_rows, accumulate, kernel):
    nothing = offsets           # stands for what is not there
    args = (lhs, rhs, out, offsets, nothing.view(torch.int32) if source is None else source, groups, rows, m, n, k, source_rows, int(bool(accumulate)), get_num_sms(),
            current_raw_stream())
    name, keys, arg_defs, code = grouped16_kernel_plan(dtype, mode, source is not None, *kernel)
    runtime = jit_tuner.compile_and_tune(name=name, keys=keys, space=(), includes=includes, arg_defs=arg_defs, template=code, args=args)
    rc = runtime(*args)
    assert rc == 0, f'{name} failed with HIP error {rc}'
    if kernel == ():
        remember_new(call, name, runtime, args)


def _m_grouped(entry, dtype, lhs, rhs, out, offsets, source, kernel=()):
    # (the entry's type is part of what a repeated call is found by: one entry's tensors are not the other's)
    call = (entry, lhs, rhs, out, offsets, source, 1 if dtype == torch.half else 0)
    if kernel == () and repeat_call(*call):
        return
    assert lhs.dim() == 2 and rhs.dim() == 3 and out.dim() == 2
    groups, n, k = rhs.shape if entry == RAGGED_NT else (rhs.size(0), rhs.size(2), rhs.size(1))
    m = out.size(0)
    _check(dtype, lhs, rhs, out, offsets, groups, source)
    assert out.dtype == dtype and out.size(1) == n and lhs.size(1) == k and m < MAX_ROWS
    assert n % 8 == 0 and k % 8 == 0 and n < MAX_COLUMNS and k < MAX_COLUMNS
    if source is None:
        assert lhs.size(0) == m
    else:
        assert source.shape == (m, ) and (lhs.size(0) > 0 or m == 0) and lhs.numel() * 2 < MAX_GATHERED_BYTES
    assert_on_current_device(lhs, rhs, out, offsets, source)
    if out.numel() == 0:
        return
    _launch(call, dtype, 'NT' if entry == RAGGED_NT else 'NN', lhs, rhs, out, offsets, source, groups, m, m, n, k, lhs.size(0), False, kernel)


def _k_grouped(dtype, lhs, rhs, out, offsets, accumulate, source, kernel=()):
    call = (RAGGED_TN, lhs, rhs, out, offsets, source, 1 if accumulate else 0, 1 if dtype == torch.half else 0)
    if kernel == () and repeat_call(*call):
        return
    assert lhs.dim() == 2 and rhs.dim() == 2 and out.dim() == 3
    groups, m, n = out.shape
    rows = lhs.size(0)
    _check(dtype, lhs, rhs, out, offsets, groups, source)
    assert out.dtype == torch.float32 and lhs.size(1) == m and rhs.size(1) == n
    assert m % 8 == 0 and n % 8 == 0 and m < MAX_COLUMNS and n < MAX_COLUMNS
    if source is None:
        assert rhs.size(0) == rows
    else:
        assert source.shape == (rows, ) and (rhs.size(0) > 0 or rows == 0) and rhs.numel() * 2 < MAX_GATHERED_BYTES
    assert_on_current_device(lhs, rhs, out, offsets, source)
    if out.numel() == 0:
        return
    if rows == 0:
        if not accumulate:
            out.zero_()
        return
    _launch(call, dtype, 'TN', lhs, rhs, out, offsets, source, groups, rows, m, n, 0, rhs.size(0), accumulate, kernel)


def m_grouped_gemm_bf16_bf16_bf16_nt_ragged(lhs: torch.Tensor, rhs: torch.Tensor, out: torch.Tensor, offsets: torch.Tensor,
                                            source: Optional[torch.Tensor] = None) -> None:
    """
    `out[r] = lhs[r] @ rhs[g].T` for the rows r of every group g, with fp32 sums.

    lhs: bf16 `[m, k]`, rhs: bf16 `[num_groups, n, k]`, out: bf16 `[m, n]`, written in place; all contiguous
    offsets: int32 `[num_groups + 1]`, ascending: group g has the rows offsets[g] .. offsets[g + 1] - 1, any number of them; rows of `out` that no group has are left as
             they were
    source: int32 `[m]`, or None: row r is `lhs[source[r]]`, lhs then having any number of rows, less than 2 GiB of them; `out[r]` is zeros where source[r] is none of them
    Requires n % 8 == 0 and k % 8 == 0; up to 1024 groups.
    """
    _m_grouped(RAGGED_NT, torch.bfloat16, lhs, rhs, out, offsets, source)


def m_grouped_gemm_fp16_fp16_fp16_nt_ragged(lhs: torch.Tensor, rhs: torch.Tensor, out: torch.Tensor, offsets: torch.Tensor,
                                            source: Optional[torch.Tensor] = None) -> None:
    """`m_grouped_gemm_bf16_bf16_bf16_nt_ragged` in fp16."""
    _m_grouped(RAGGED_NT, torch.half, lhs, rhs, out, offsets, source)


def m_grouped_gemm_bf16_bf16_bf16_nn_ragged(lhs: torch.Tensor, rhs: torch.Tensor, out: torch.Tensor, offsets: torch.Tensor) -> None:
    """
    `out[r] = lhs[r] @ rhs[g]` for the rows r of every group g: the gradient of the rows, with the weights as the forward product has them.

    lhs: bf16 `[m, k]`, rhs: bf16 `[num_groups, k, n]`, out: bf16 `[m, n]`; the rest as for `m_grouped_gemm_bf16_bf16_bf16_nt_ragged`
    """
    _m_grouped(RAGGED_NN, torch.bfloat16, lhs, rhs, out, offsets, None)


def m_grouped_gemm_fp16_fp16_fp16_nn_ragged(lhs: torch.Tensor, rhs: torch.Tensor, out: torch.Tensor, offsets: torch.Tensor) -> None:
    """`m_grouped_gemm_bf16_bf16_bf16_nn_ragged` in fp16."""
    _m_grouped(RAGGED_NN, torch.half, lhs, rhs, out, offsets, None)


def k_grouped_gemm_bf16_bf16_fp32_tn_ragged(lhs: torch.Tensor, rhs: torch.Tensor, out: torch.Tensor, offsets: torch.Tensor, accumulate: bool = False,
                                            source: Optional[torch.Tensor] = None) -> None:
    """
    `out[g] = lhs[rows of g].T @ rhs[rows of g]`, or `+=` with `accumulate`: the gradients of all experts' weights, in fp32.

    lhs: bf16 `[rows, m]`, the gradients of the outputs; rhs: bf16 `[rows, n]`, the inputs; out: fp32 `[num_groups, m, n]`, written in place; all contiguous
    offsets: as for `m_grouped_gemm_bf16_bf16_bf16_nt_ragged`, of the rows; a group without rows is zero, or unchanged with `accumulate`
    source: int32 `[rows]`, or None: the input of row r is `rhs[source[r]]`, rhs then having any number of rows, less than 2 GiB of them; a row whose source[r] is none of them
            counts for nothing, whatever lhs[r] holds
    Requires m % 8 == 0 and n % 8 == 0; up to 1024 groups.
    """
    _k_grouped(torch.bfloat16, lhs, rhs, out, offsets, accumulate, source)


def k_grouped_gemm_fp16_fp16_fp32_tn_ragged(lhs: torch.Tensor, rhs: torch.Tensor, out: torch.Tensor, offsets: torch.Tensor, accumulate: bool = False,
                                            source: Optional[torch.Tensor] = None) -> None:
    """`k_grouped_gemm_bf16_bf16_fp32_tn_ragged` of fp16 operands."""
    _k_grouped(torch.half, lhs, rhs, out, offsets, accumulate, source)
