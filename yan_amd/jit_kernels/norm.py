"""Root-mean-square norm in front of the GEMMs: the residual's addition, the norm and the FP8 quantiser in one kernel, and its gradient.

The reference's FP8 entry takes quantised activations (`lhs, lhs_scales`, `yan/jit_kernels/gemm.py:23-30`) and has nothing that makes them; in a model they come
out of a norm. `rms_norm_to_fp8` leaves what `per_token_cast_to_fp8` of the normed rows would, without the trip through memory (and without the rounding to 16
bits in between); `rms_norm` is the same for the 16-bit GEMMs. Both add the residual first where there is one:

    h = x + residual, rounded to the residual's type and stored in its place;   r = (mean(h^2) + eps)^-1/2;   y = h * r * weight

`rms_norm_backward` gives the gradient of h, which is that of x and of the residual, and of the weight.
"""
import functools
from typing import Optional, Tuple

import torch

from .host_calls import NORM, NORM_BACKWARD, remember_new, repeat_new
from .tuner import FrozenKeys, jit_tuner
from .utils import assert_on_current_device, ceil_div, current_raw_stream

includes = ('"norm/rms_norm.hpp"', )

# kNormMostColumns of norm/rms_norm.hpp
MAX_COLUMNS = 16384
_ELEMENTS = {torch.bfloat16: '__bf16', torch.float32: 'float'}

template = """
using namespace yan;
// Templated args from Python JIT call: {X} + {H} (added: {RESIDUAL}) times {W}; {LANES} lanes a row with {RUNS} runs of 8 each; codes {CODES}, 16 bits {NORMED}
__return_code = static_cast<int>(launch_rms_norm<{X}, {H}, {W}, {LANES}, {RUNS}, {RESIDUAL}, {CODES}, {NORMED}>(
    reinterpret_cast<const {X}*>(x), reinterpret_cast<{H}*>(residual), reinterpret_cast<const {W}*>(weight), codes, scales, stride_m, stride_k, normed, inverse_rms,
    rows, k, eps, stream));
"""

backward_template = """
using namespace yan;
// Templated args from Python JIT call: gradients {G}, h {H}, weight {W}; {LANES} lanes a row with {RUNS} runs of 8 each; a residual's gradient {RESIDUAL}, the weight's {WEIGHT}
__return_code = static_cast<int>(launch_rms_norm_backward<{G}, {H}, {W}, {LANES}, {RUNS}, {RESIDUAL}, {WEIGHT}>(
    reinterpret_cast<const {G}*>(grad), reinterpret_cast<const {H}*>(h), reinterpret_cast<const {W}*>(weight), inverse_rms, reinterpret_cast<const {G}*>(grad_residual),
    reinterpret_cast<{G}*>(grad_h), partial, workgroups, grad_weight, accumulate != 0, rows, k, stream));
"""


def _arg_defs(x, h, w):
    return (('x', x), ('weight', w), ('residual', h), ('normed', torch.bfloat16), ('codes', torch.float8_e4m3fn), ('scales', torch.float), ('inverse_rms', torch.float),
            ('stride_m', int), ('stride_k', int), ('rows', int), ('k', int), ('eps', float), ('stream', torch.cuda.Stream))


def _backward_arg_defs(g, h, w):
    return (('grad', g), ('h', h), ('weight', w), ('inverse_rms', torch.float), ('grad_weight', torch.float), ('grad_residual', g), ('grad_h', g),
            ('partial', torch.float), ('workgroups', int), ('accumulate', int), ('rows', int), ('k', int), ('stream', torch.cuda.Stream))


def norm_lanes(rows: int, k: int) -> Tuple[int, int]:
    """(lanes a row, runs of 8 elements a lane) of the norm's kernel."""
    runs = ceil_div(k, 8)
    for lanes, most in ((16, 2), (64, 4), (256, 8)):
        if runs <= lanes * (1 if rows <= 1024 else most):
            break
    else:
        lanes = 1024
    each = ceil_div(runs, lanes)
    return lanes, 1 if each == 1 else 2 if each == 2 else 4 if each <= 4 else 8


def norm_backward_lanes(k: int) -> Tuple[int, int]:
    """
    The same of its gradient's, where a lane has two rows (up to 256 lanes) and the weight's sums in its registers. Wider rows one at a time on 1024 lanes (8192 x 16384
    200 us; two of them on 512 lanes do not fit the registers: 317), which leaves 20 bytes of a lane in scratch where h and the weight are fp32 and both gradients are asked for.
    """
    runs = ceil_div(k, 8)
    for lanes in (16, 64, 256, 1024):
        if runs <= lanes * (2 if lanes == 16 else 4):
            break
    each = ceil_div(runs, lanes)
    return lanes, 1 if each == 1 else 2 if each == 2 else 4


def norm_backward_workgroups(rows: int, k: int) -> int:
    """
    Workgroups of the gradient's kernel, each of which leaves its sums of the weight's gradient, to be added up behind it: one a compute unit where the rows that it has
    in flight are enough to keep it busy (us with 256 and with 512: 8192 x 7168 92.7, 97.4; 1023 x 7168 16.4, 20.6; 8192 x 16384 200, 207; 32768 x 1024, four rows at a
    time, 45.7, 49.8), two where they are not (4096 x 2112 19.7, 16.4).
    """
    lanes, _ = norm_backward_lanes(k)
    at_a_time = max(1, 256 // lanes)
    return max(1, min(ceil_div(rows, at_a_time), 256 if at_a_time * k >= 4096 else 512))


@functools.lru_cache(maxsize=None)
def norm_kernel_plan(x: torch.dtype, h: torch.dtype, w: torch.dtype, lanes: int, runs: int, residual: bool, codes: bool, normed: bool):
    """(name, keys, arg_defs, template) of the norm's kernel; needs no GPU."""
    yes = {False: 'false', True: 'true'}
    keys = FrozenKeys({'X': _ELEMENTS[x], 'H': _ELEMENTS[h], 'W': _ELEMENTS[w], 'LANES': lanes, 'RUNS': runs, 'RESIDUAL': yes[residual], 'CODES': yes[codes],
                       'NORMED': yes[normed]})
    return 'rms_norm', keys, _arg_defs(x, h, w), template


@functools.lru_cache(maxsize=None)
def norm_backward_kernel_plan(g: torch.dtype, h: torch.dtype, w: torch.dtype, lanes: int, runs: int, residual: bool, weight: bool):
    """(name, keys, arg_defs, template) of the gradient's kernels; needs no GPU."""
    yes = {False: 'false', True: 'true'}
    keys = FrozenKeys({'G': _ELEMENTS[g], 'H': _ELEMENTS[h], 'W': _ELEMENTS[w], 'LANES': lanes, 'RUNS': runs, 'RESIDUAL': yes[residual], 'WEIGHT': yes[weight]})
    return 'rms_norm_backward', keys, _backward_arg_defs(g, h, w), backward_template


def _check(x, weight, *others):
    assert x.dim() == 2 and x.dtype in _ELEMENTS and x.is_contiguous() and x.size(0) < 1 << 31
    assert 0 < x.size(1) <= MAX_COLUMNS and x.size(1) % 8 == 0, 'rows of up to 16384 elements, a multiple of 8'
    assert weight.shape == (x.size(1), ) and weight.dtype in _ELEMENTS and weight.is_contiguous()
    for t in (x, weight, *others):
        assert t is None or t.data_ptr() % 16 == 0, 'tensors start at multiples of 16 bytes'
    for t in others:
        assert t is None or (t.shape == x.shape and t.dtype in _ELEMENTS and t.is_contiguous())


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share no byte, whatever they are views of (tensors without memory have address 0). 0.3 us."""
    ahead = b.data_ptr() - a.data_ptr()
    if ahead:
        return ahead >= a.nbytes if ahead > 0 else -ahead >= b.nbytes
    return not a.data_ptr() or not a.nbytes or not b.nbytes


def _run(plan, args):
    name, keys, arg_defs, code = plan
    runtime = jit_tuner.compile_and_tune(name=name, keys=keys, space=(), includes=includes, arg_defs=arg_defs, template=code, args=args)
    rc = runtime(*args)
    assert rc == 0, f'{name} failed with HIP error {rc}'
    return name, runtime, args


def _norm(call, x, weight, eps, residual, col_major_scales, normed, with_codes):
    _check(x, weight, residual, normed)
    assert normed is None or normed.dtype == torch.bfloat16
    assert not with_codes or x.size(1) % 128 == 0, 'a scale covers 128 elements'
    assert_on_current_device(x, weight, residual, normed)
    rows, k = x.shape
    inverse_rms = torch.empty((rows, ), dtype=torch.float32, device=x.device)
    codes = scales = None
    if with_codes:
        codes = torch.empty((rows, k), dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty((k // 128, rows), dtype=torch.float32, device=x.device).t() if col_major_scales else torch.empty((rows, k // 128), dtype=torch.float32, device=x.device)
    made = (codes, scales, inverse_rms) if with_codes else (inverse_rms, )
    if rows == 0:
        return made
    nothing = inverse_rms           # stands for what is not there
    h = x.dtype if residual is None else residual.dtype
    done = _run(norm_kernel_plan(x.dtype, h, weight.dtype, *norm_lanes(rows, k), residual is not None, with_codes, normed is not None),
                (x, weight, nothing.view(h) if residual is None else residual, nothing.view(torch.bfloat16) if normed is None else normed,
                 nothing.view(torch.float8_e4m3fn) if codes is None else codes, nothing if scales is None else scales, inverse_rms,
                 *(scales.stride() if with_codes else (0, 0)), rows, k, float(eps), current_raw_stream()))
    remember_new(call, *done, made)
    return made


def rms_norm_to_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None, col_major_scales: bool = False,
                    normed: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    The normed rows as an operand of the FP8 GEMMs.

    x: bf16 or fp32 `[m, k]`, contiguous, k % 128 == 0, k up to 16384; weight: bf16 or fp32 `[k]`
    residual: bf16 or fp32 `[m, k]` (of x's type or not), or None: becomes `x + residual`, which is what is normed
    normed: bf16 `[m, k]`, or None: gets the normed rows in 16 bits as well (for a router); may be x itself, no part of the residual
    Returns e4m3fn `[m, k]` and fp32 scales `[m, k/128]`, as `per_token_cast_to_fp8` makes them of the normed rows in fp32 (with `col_major_scales`
    token-contiguous), and fp32 `[m]`, the reciprocals of the root mean squares, for the gradient. Squares are summed in fp32.
    """
    # (no part of what a repeated call is found by)
    assert eps >= 0
    assert normed is None or residual is None or (normed is not residual and _apart(normed, residual)), 'the normed rows have a place of their own'
    call = (NORM, x, weight, residual, normed, float(eps), 2 if col_major_scales else 1)
    made = repeat_new(*call)
    if made is not None:
        return made
    return _norm(call, x, weight, eps, residual, col_major_scales, normed, True)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    The normed rows in 16 bits: out bf16 `[m, k]`, written in place (may be x itself, no part of the residual), k % 8 == 0; the rest as for `rms_norm_to_fp8`. Returns the reciprocals of the root mean
    squares, fp32 `[m]`.
    """
    assert eps >= 0
    assert out is not None and (residual is None or (out is not residual and _apart(out, residual))), 'the normed rows have a place of their own'
    call = (NORM, x, weight, residual, out, float(eps), 0)
    made = repeat_new(*call)
    if made is not None:
        return made[0]
    return _norm(call, x, weight, eps, residual, False, out, False)[0]


def rms_norm_backward(grad_out: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, inverse_rms: torch.Tensor, grad_weight: Optional[torch.Tensor] = None,
                      grad_residual: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """
    The gradient of h, that is of x and of the residual, of `rms_norm` and `rms_norm_to_fp8` (whose codes' roundings count as the identity).

    grad_out: bf16 or fp32 `[m, k]`, contiguous: the gradient of the normed rows
    h: bf16 or fp32 `[m, k]`: what was normed, the residual as the call left it, or x; weight, inverse_rms: as given and returned there
    grad_weight: fp32 `[k]`, written in place, or added to with `accumulate`; None: not wanted
    grad_residual: `[m, k]` of grad_out's type, or None: what reaches h from elsewhere, added to the result
    Returns the gradient in grad_out's type. Results repeat to the bit.
    """
    call = (NORM_BACKWARD, grad_out, h, weight, inverse_rms, grad_weight, grad_residual, 1 if accumulate else 0)
    made = repeat_new(*call)
    if made is not None:
        return made[0]
    _check(grad_out, weight, h, grad_residual)
    rows, k = grad_out.shape
    assert inverse_rms.shape == (rows, ) and inverse_rms.dtype == torch.float32 and inverse_rms.is_contiguous()
    assert grad_residual is None or grad_residual.dtype == grad_out.dtype
    if grad_weight is not None:
        assert grad_weight.shape == (k, ) and grad_weight.dtype == torch.float32 and grad_weight.is_contiguous()
    assert_on_current_device(grad_out, h, weight, inverse_rms, grad_weight, grad_residual)
    grad_h = torch.empty_like(grad_out)
    if rows == 0:
        if grad_weight is not None and not accumulate:
            grad_weight.zero_()
        return grad_h
    lanes, runs = norm_backward_lanes(k)
    workgroups = norm_backward_workgroups(rows, k)
    partial = None if grad_weight is None else torch.empty((workgroups * max(1, 256 // lanes), k), dtype=torch.float32, device=h.device)
    nothing = inverse_rms           # stands for what is not there
    done = _run(norm_backward_kernel_plan(grad_out.dtype, h.dtype, weight.dtype, lanes, runs, grad_residual is not None, grad_weight is not None),
                (grad_out, h, weight, inverse_rms, nothing if grad_weight is None else grad_weight, nothing.view(grad_out.dtype) if grad_residual is None else grad_residual,
                 grad_h, nothing if partial is None else partial, workgroups, int(bool(accumulate)), rows, k, current_raw_stream()))
    remember_new(call, *done, (grad_h, ), () if partial is None else (partial, ))
    return grad_h
