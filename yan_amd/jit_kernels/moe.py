"""Around the grouped (expert) FP8 GEMMs: the router with its balance loss, tokens to the experts' rows, and back.

The reference has the grouped layouts' hooks (`yan/include/gemm/scheduler.cuh:7-11,31-48`, `yan/jit_kernels/utils.py:46-55`) and nothing that
fills the layouts or empties them; callers of `m_grouped_gemm_fp8_fp8_bf16_nt_*` type chains of torch ops for it. A forward pass here:

    weights, indices, counts, loss = moe_route(logits, top_k)
    rows, m_indices, source, offsets = moe_dispatch_to_fp8_contiguous(x, indices, num_experts, (x8, scales))
    m_grouped_gemm_fp8_fp8_bf16_nt_contiguous((x8, scales), experts, y, m_indices)
    moe_combine(y, rows, weights, out)

and back: `moe_combine_backward`, `per_channel_cast_to_fp8` of both sides and `k_grouped_gemm_fp8_fp8_fp32_nt_contiguous` for the experts' weights,
`moe_combine` without weights for the tokens' gradients, `moe_route_backward` for the logits. Work is enqueued on the current stream; what the
entries return is allocated from torch's caching allocator, and so is the scratch of a call. The router's workgroups for few tokens meet in the
stream's split-K workspace (`split_k.py`), unless `YAN_SPLIT_K=0`.
"""
import functools
from typing import Optional, Tuple

import torch

from .host_calls import COMBINE, COMBINE_BACKWARD, DISPATCH, LAYOUT, ROUTE, ROUTE_BACKWARD, remember_new, repeat_call, repeat_new
from .split_k import split_k_launch_failed, split_k_workspace
from .tuner import FrozenKeys, jit_tuner
from .utils import assert_on_current_device, ceil_div, current_raw_stream, get_m_alignment_for_contiguous_layout

# kMaxTopK, kMaxTokens and kMaxExperts of moe/route.hpp, kFewPairs, kTokensPerBlock and kMaxPairs of moe/dispatch.hpp
MAX_TOP_K = 16
MAX_TOKENS = 1 << 30
MAX_EXPERTS = 1024
FEW_PAIRS = 4096
TOKENS_PER_BLOCK = 16
MAX_PAIRS = (1 << 31) - (1 << 18)
# kLayoutChunk and kLayoutFewChunks of moe/layout.hpp
LAYOUT_CHUNK = 1024
LAYOUT_FEW_CHUNKS = 8

_ELEMENTS = {torch.bfloat16: '__bf16', torch.float32: 'float'}
_SCORINGS = {'softmax': 0, 'sigmoid': 1}


def _run(plan, includes, args, token=None):
    name, keys, arg_defs, template = plan
    runtime = jit_tuner.compile_and_tune(name=name, keys=keys, space=(), includes=includes, arg_defs=arg_defs, template=template, args=args)
    rc = runtime(*args)
    if rc != 0 and token is not None:
        split_k_launch_failed(token)
    assert rc == 0, f'{name} failed with HIP error {rc}'
    return name, runtime, args


# Router

_route_includes = ('"moe/route.hpp"', )

route_template = """
using namespace yan;
// Templated args from Python JIT call: element {ELEMENT} of the logits, sigmoid {SIGMOID}, {LANES} lanes a token with {VALUES} logits each, {THREADS} threads a workgroup
__return_code = static_cast<int>(launch_moe_route<{ELEMENT}, {SIGMOID}, {LANES}, {VALUES}, {THREADS}>(
    reinterpret_cast<const {ELEMENT}*>(logits), masked ? mask : nullptr, weights, indices, counts, loss, workspace, blocks, join != 0, tokens, experts, top_k,
    renormalize != 0, stream));
"""

route_backward_template = """
using namespace yan;
// Templated args from Python JIT call: element {ELEMENT} of the logits, sigmoid {SIGMOID}, {LANES} lanes a token with {VALUES} logits each
__return_code = static_cast<int>(launch_moe_route_backward<{ELEMENT}, {SIGMOID}, {LANES}, {VALUES}>(
    reinterpret_cast<const {ELEMENT}*>(logits), indices, counts, has_weights ? grad_weights : nullptr, has_loss ? grad_loss : nullptr,
    reinterpret_cast<{ELEMENT}*>(grad_logits), tokens, experts, top_k, renormalize != 0, stream));
"""


def _route_arg_defs(dtype):
    return (('logits', dtype), ('mask', torch.uint8), ('weights', torch.float), ('indices', torch.int), ('counts', torch.int), ('loss', torch.float),
            ('workspace', torch.uint8), ('masked', int), ('blocks', int), ('join', int), ('tokens', int), ('experts', int), ('top_k', int), ('renormalize', int),
            ('stream', torch.cuda.Stream))


def _route_backward_arg_defs(dtype):
    return (('logits', dtype), ('indices', torch.int), ('counts', torch.int), ('grad_weights', torch.float), ('grad_loss', torch.float),
            ('grad_logits', dtype), ('has_weights', int), ('has_loss', int), ('tokens', int), ('experts', int), ('top_k', int), ('renormalize', int),
            ('stream', torch.cuda.Stream))


def route_lanes(experts: int) -> Tuple[int, int]:
    """(lanes a token, logits a lane) of the router's kernels."""
    if experts <= 64:
        return 16, 4
    for lanes, values in ((32, 4), (64, 4), (64, 8)):
        if experts <= lanes * values:
            return lanes, values
    return 64, 16


def route_threads(tokens: int, experts: int) -> int:
    """Threads of a workgroup of the router's kernel: few, so that few tokens are spread over many compute units, as long as that leaves no more
    rows of counts and shares to add up than 256. One token of 256 experts takes 4.0 us in 256 threads and 5.5 in 1024, one of 1024 experts 27 and 11."""
    return 256 if experts <= 512 and ceil_div(tokens, 256 // route_lanes(experts)[0]) <= 256 else 1024


def route_blocks(tokens: int, experts: int) -> int:
    """Workgroups of the router's kernel; one alone has nothing to add up."""
    at_once = route_threads(tokens, experts) // route_lanes(experts)[0]
    return min(max(1, ceil_div(tokens, at_once)), 256)


def route_joins(blocks: int, experts: int) -> bool:
    """Whether the last of the workgroups adds up all their rows. 64 tokens of 256 experts, 16 workgroups: 6.5 us on the device instead of 7.7 with a second
    kernel, 5.9 a call instead of 7.8; 256 tokens, 64 workgroups: 8.6 instead of 8.1; 1024 tokens, 256 workgroups: 19.8 instead of 9.4. In two levels of 16: 10.4."""
    return 1 < blocks <= 64 and blocks * experts <= 8192


@functools.lru_cache(maxsize=None)
def route_kernel_plan(dtype: torch.dtype, scoring: str, experts: int, backward: bool = False, threads: int = 256):
    """(name, keys, arg_defs, template) of the router's kernel, forward in workgroups of `threads`; needs no GPU. The same for all `experts` with the same
    `route_lanes`."""
    lanes, values = route_lanes(experts)
    keys = {'ELEMENT': _ELEMENTS[dtype], 'SIGMOID': 'true' if scoring == 'sigmoid' else 'false', 'LANES': lanes, 'VALUES': values}
    if backward:
        return 'moe_route_backward', FrozenKeys(keys), _route_backward_arg_defs(dtype), route_backward_template
    return 'moe_route', FrozenKeys({**keys, 'THREADS': threads}), _route_arg_defs(dtype), route_template


def _check_route(logits, top_k, scoring):
    assert logits.dim() == 2 and logits.dtype in _ELEMENTS and logits.is_contiguous() and logits.size(0) <= MAX_TOKENS
    assert 1 <= logits.size(1) <= MAX_EXPERTS and 1 <= top_k <= min(MAX_TOP_K, logits.size(1))
    assert scoring in ('softmax', 'sigmoid')


def moe_route(logits: torch.Tensor, top_k: int, scoring: str = 'softmax', renormalize: bool = True,
              mask: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    The `top_k` experts of every token with their weights, the number of tokens of every expert, and the balance loss.

    logits: bf16 or fp32 `[tokens, experts]`, contiguous; up to 1024 experts, top_k up to 16
    scoring: scores s are 'softmax' or 'sigmoid' of the logits
    renormalize: weights are s over the sum of s of the token's picks; else s itself (0 for sigmoid scores below 2^-126)
    mask: bool `[tokens]`; tokens where it is false are padding: indices -1, weights 0, in neither counts nor loss
    Returns weights fp32 `[tokens, top_k]`, indices int32 `[tokens, top_k]` (largest logit first, ties to the lowest expert), counts int32
    `[experts]` and loss, fp32 with no dimensions: `experts * sum_e f_e P_e`, f_e the share of the picks that are e and P_e the mean over the tokens
    of s (softmax) or of s over the row's sum of s (sigmoid); 0 when no token counts. Results repeat to the bit.
    Logits of -infinity are picked after all others, with weight 0, and +infinity counts as the largest finite number. A NaN makes its token's
    weights and the loss NaN.
    """
    call = (ROUTE, logits, mask, top_k, _SCORINGS.get(scoring, -1), 1 if renormalize else 0)
    made = repeat_new(*call)
    if made is not None:
        return made
    _check_route(logits, top_k, scoring)
    tokens, experts = logits.shape
    if mask is not None:
        assert mask.shape == (tokens, ) and mask.dtype == torch.bool and mask.is_contiguous()
    assert_on_current_device(logits, mask)
    device = logits.device
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
    indices = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
    counts = torch.empty((experts, ), dtype=torch.int32, device=device)
    loss = torch.empty((), dtype=torch.float32, device=device)
    threads, blocks = route_threads(tokens, experts), route_blocks(tokens, experts)
    stream = current_raw_stream()
    # the workgroups' counts and shares: joined within the kernel, in the split-K workspace of the stream, or left in scratch for a second one
    joined, token = split_k_workspace(device, stream) if route_joins(blocks, experts) else (None, None)
    # RouteWorkspace::bytes of moe/route.hpp
    scratch = None if joined is not None or blocks == 1 else torch.empty(4 * (2 * blocks * experts + 3 * ceil_div(experts, 16) + 1), dtype=torch.uint8, device=device)
    workspace = joined if joined is not None else scratch if scratch is not None else weights.view(torch.uint8)
    mask_bytes = workspace if mask is None else mask.view(torch.uint8)
    done = _run(route_kernel_plan(logits.dtype, scoring, experts, False, threads), _route_includes,
                (logits, mask_bytes, weights, indices, counts, loss, workspace, int(mask is not None), blocks, int(joined is not None), tokens, experts, top_k,
                 int(bool(renormalize)), stream), token)
    made = (weights, indices, counts, loss)
    remember_new(call, *done, made, () if scratch is None else (scratch, ), {} if mask is None else {id(mask_bytes): mask}, joined)
    return made


def moe_route_backward(logits: torch.Tensor, indices: torch.Tensor, counts: torch.Tensor, grad_weights: Optional[torch.Tensor],
                       grad_loss: Optional[torch.Tensor], scoring: str = 'softmax', renormalize: bool = True) -> torch.Tensor:
    """
    The gradient of the logits of `moe_route`, in their type, from what the call was given and returned.

    grad_weights: fp32 `[tokens, top_k]`, or None for zero; grad_loss: fp32 with one element, on the device, or None for zero
    The picks and `counts` are constants of the loss. Masked tokens (indices -1) get zeros.
    """
    call = (ROUTE_BACKWARD, logits, indices, counts, grad_weights, grad_loss, _SCORINGS.get(scoring, -1), 1 if renormalize else 0)
    made = repeat_new(*call)
    if made is not None:
        return made[0]
    assert indices.dim() == 2
    top_k = indices.size(1)
    _check_route(logits, top_k, scoring)
    tokens, experts = logits.shape
    assert indices.shape == (tokens, top_k) and indices.dtype == torch.int32 and indices.is_contiguous()
    assert counts.shape == (experts, ) and counts.dtype == torch.int32 and counts.is_contiguous()
    if grad_weights is not None:
        assert grad_weights.shape == (tokens, top_k) and grad_weights.dtype == torch.float32 and grad_weights.is_contiguous()
    if grad_loss is not None:
        assert grad_loss.numel() == 1 and grad_loss.dtype == torch.float32
    assert_on_current_device(logits, indices, counts, grad_weights, grad_loss)
    grad_logits = torch.empty_like(logits)
    if tokens == 0:
        return grad_logits
    nothing = torch.empty(1, dtype=torch.float32, device=logits.device)         # stands for what is not there
    done = _run(route_kernel_plan(logits.dtype, scoring, experts, True), _route_includes,
                (logits, indices, counts, nothing if grad_weights is None else grad_weights, nothing if grad_loss is None else grad_loss, grad_logits,
                 int(grad_weights is not None), int(grad_loss is not None), tokens, experts, top_k, int(bool(renormalize)), current_raw_stream()))
    remember_new(call, *done, (grad_logits, ))
    return grad_logits


# Tokens to the experts' rows

_dispatch_includes = ('"moe/dispatch.hpp"', )

dispatch_template = """
using namespace yan;
// Templated args from Python JIT call: element {ELEMENT} of the activations
__return_code = static_cast<int>(launch_moe_dispatch(
    reinterpret_cast<const {ELEMENT}*>(x), indices, codes, scales, stride_g, stride_m, stride_k, rows_of, m_indices, source, offsets, workspace, workspace_bytes,
    tokens, k, top_k, experts, m_max, rows, stream));
"""


def _dispatch_arg_defs(dtype):
    return (('x', dtype), ('indices', torch.int), ('codes', torch.float8_e4m3fn), ('scales', torch.float), ('rows_of', torch.int), ('m_indices', torch.int),
            ('source', torch.int), ('offsets', torch.int), ('workspace', torch.uint8), ('workspace_bytes', int), ('stride_g', int), ('stride_m', int),
            ('stride_k', int), ('tokens', int), ('k', int), ('top_k', int), ('experts', int), ('m_max', int), ('rows', int), ('stream', torch.cuda.Stream))


@functools.lru_cache(maxsize=None)
def dispatch_kernel_plan(dtype: torch.dtype):
    """(name, keys, arg_defs, template) of the dispatch kernel; needs no GPU."""
    return 'moe_dispatch_to_fp8', FrozenKeys({'ELEMENT': _ELEMENTS[dtype]}), _dispatch_arg_defs(dtype), dispatch_template


def get_contiguous_layout_rows(num_tokens: int, top_k: int, num_experts: int) -> int:
    """Rows that the contiguous layout of `num_tokens * top_k` pairs takes at most, however they fall on the experts."""
    pairs, alignment = num_tokens * top_k, get_m_alignment_for_contiguous_layout()
    return (pairs + (alignment - 1) * min(num_experts, pairs)) // alignment * alignment


def _check_dispatch(x, indices, codes, scales, num_experts):
    assert x.dim() == 2 and x.dtype in _ELEMENTS and x.is_contiguous() and x.size(1) % 128 == 0 and x.size(1) > 0
    assert indices.dim() == 2 and indices.size(0) == x.size(0) and indices.dtype == torch.int32 and indices.is_contiguous()
    assert 1 <= indices.size(1) <= MAX_TOP_K and 1 <= num_experts <= MAX_EXPERTS and indices.numel() <= MAX_PAIRS
    assert codes.dtype == torch.float8_e4m3fn and codes.is_contiguous() and codes.size(-1) == x.size(1)
    assert scales.dtype == torch.float32 and scales.shape == (*codes.shape[:-1], x.size(1) // 128)
    assert codes.numel() // x.size(1) < 1 << 31 and all(0 <= s < 1 << 31 for s in scales.stride())
    assert x.data_ptr() % 16 == 0 and codes.data_ptr() % 16 == 0, 'activations and codes start at multiples of 16 bytes'


def _dispatch(call, x, indices, codes, scales, num_experts, m_max, made):
    # `made`: rows and masked_m of the masked layout; rows, m_indices, source and offsets of the contiguous one
    tokens, k = x.shape
    top_k, rows = indices.size(1), codes.numel() // k
    few = tokens * top_k <= FEW_PAIRS
    # moe_dispatch_workspace_bytes of moe/dispatch.hpp
    workspace_bytes = 0 if few else (ceil_div(tokens, TOKENS_PER_BLOCK) + 1) * num_experts * 4
    assert workspace_bytes < 1 << 31
    scratch = None if few else torch.empty(workspace_bytes, dtype=torch.uint8, device=x.device)
    workspace = made[0].view(torch.uint8) if few else scratch           # no call with few pairs looks at it
    strides = scales.stride() if m_max else (0, *scales.stride())
    rows_of, m_indices, source, offsets = made if not m_max else (made[0], made[1], made[1], made[1])
    done = _run(dispatch_kernel_plan(x.dtype), _dispatch_includes,
                (x, indices, codes, scales, rows_of, m_indices, source, offsets, workspace, workspace_bytes, *strides, tokens, k, top_k, num_experts, m_max, rows,
                 current_raw_stream()))
    remember_new(call, *done, made, () if few else (scratch, ))
    return made


def moe_dispatch_to_fp8_contiguous(x: torch.Tensor, indices: torch.Tensor, num_experts: int,
                                   out: Tuple[torch.Tensor, torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    Every (token, pick) quantised into a row of its expert, in the layout of `m_grouped_gemm_fp8_fp8_bf16_nt_contiguous`.

    x: bf16 or fp32 `[tokens, k]`, contiguous, k % 128 == 0
    indices: int32 `[tokens, top_k]`, the experts of every token; others than 0 .. num_experts - 1 (-1 of a masked token) go nowhere
    out: (e4m3fn `[m_sum, k]` contiguous, fp32 scales `[m_sum, k/128]` in any strided layout), written in place with the bits of
         `per_token_cast_to_fp8`; rows that no pair has are left as they were. m_sum is a multiple of
         `get_m_alignment_for_contiguous_layout()`; `get_contiguous_layout_rows` is always enough, and pairs past it get no row.
    Returns rows int32 `[tokens, top_k]` (the row of every pair, -1: none), m_indices int32 `[m_sum]` for the GEMM, source int32 `[m_sum]` (the token
    of every row, -1: none) and offsets int32 `[num_experts + 1]` (where every expert's rows start). An expert's rows are in the order of
    (token, pick).
    """
    codes, scales = out
    call = (DISPATCH, x, indices, codes, scales, num_experts)
    made = repeat_new(*call)
    if made is not None:
        return made
    _check_dispatch(x, indices, codes, scales, num_experts)
    m_sum = codes.size(0)
    assert codes.dim() == 2 and m_sum % get_m_alignment_for_contiguous_layout() == 0
    assert_on_current_device(x, indices, codes, scales)
    device = x.device
    rows = torch.empty_like(indices)
    m_indices = torch.empty((m_sum, ), dtype=torch.int32, device=device)
    source = torch.empty((m_sum, ), dtype=torch.int32, device=device)
    offsets = torch.empty((num_experts + 1, ), dtype=torch.int32, device=device)
    return _dispatch(call, x, indices, codes, scales, num_experts, 0, (rows, m_indices, source, offsets))


def moe_dispatch_to_fp8_masked(x: torch.Tensor, indices: torch.Tensor, out: Tuple[torch.Tensor, torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    The same into the layout of `m_grouped_gemm_fp8_fp8_bf16_nt_masked`: every expert owns `m_max` rows.

    out: (e4m3fn `[num_experts, m_max, k]` contiguous, fp32 scales `[num_experts, m_max, k/128]` in any strided layout)
    Returns rows int32 `[tokens, top_k]` (expert * m_max + place; -1 for a pair past its expert's m_max rows, the later ones in the order of (token, pick))
    and masked_m int32 `[num_experts]`, the rows that every expert has.
    """
    codes, scales = out
    call = (DISPATCH, x, indices, codes, scales)
    made = repeat_new(*call)
    if made is not None:
        return made
    assert codes.dim() == 3 and codes.size(1) > 0
    num_experts, m_max, _ = codes.shape
    _check_dispatch(x, indices, codes, scales, num_experts)
    assert_on_current_device(x, indices, codes, scales)
    rows = torch.empty_like(indices)
    masked_m = torch.empty((num_experts, ), dtype=torch.int32, device=x.device)
    return _dispatch(call, x, indices, codes, scales, num_experts, m_max, (rows, masked_m))


# The same rows without padding and without copies of the tokens, for the 16-bit products

_layout_includes = ('"moe/layout.hpp"', )

layout_template = """
using namespace yan;
__return_code = static_cast<int>(launch_moe_layout(indices, rows, source, offsets, workspace, workspace_numbers, pairs, top_k, experts, stream));
"""
layout_arg_defs = (('indices', torch.int), ('rows', torch.int), ('source', torch.int), ('offsets', torch.int), ('workspace', torch.int), ('workspace_numbers', int),
                   ('pairs', int), ('top_k', int), ('experts', int), ('stream', torch.cuda.Stream))


@functools.lru_cache(maxsize=None)
def layout_kernel_plan():
    """(name, keys, arg_defs, template) of the ragged layout's kernels; needs no GPU."""
    return 'moe_ragged_layout', FrozenKeys({}), layout_arg_defs, layout_template


def moe_ragged_layout(indices: torch.Tensor, num_experts: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    The rows of every expert right behind those of the one before it: the layout of `m_grouped_gemm_bf16_bf16_bf16_nt_ragged`, which gathers its rows itself.

    indices: int32 `[tokens, top_k]`, the experts of every token; others than 0 .. num_experts - 1 (-1 of a masked token) have no row
    Returns rows int32 `[tokens, top_k]` (the row of every pair, -1: none), source int32 `[tokens * top_k]` (the token of every row, -1 behind the last one) and
    offsets int32 `[num_experts + 1]` (where every expert's rows start, and where the last one's end). An expert's rows are in the order of (token, pick).
    """
    call = (LAYOUT, indices, num_experts)
    made = repeat_new(*call)
    if made is not None:
        return made
    assert indices.dim() == 2 and indices.dtype == torch.int32 and indices.is_contiguous()
    assert 1 <= indices.size(1) <= MAX_TOP_K and 1 <= num_experts <= MAX_EXPERTS and indices.numel() <= MAX_PAIRS
    assert_on_current_device(indices)
    device, pairs = indices.device, indices.numel()
    rows = torch.empty_like(indices)
    source = torch.empty((pairs, ), dtype=torch.int32, device=device)
    offsets = torch.empty((num_experts + 1, ), dtype=torch.int32, device=device)
    # moe_layout_workspace_numbers of moe/layout.hpp
    chunks = ceil_div(pairs, LAYOUT_CHUNK)
    numbers = 0 if chunks <= LAYOUT_FEW_CHUNKS else (chunks + 1) * num_experts
    scratch = torch.empty(numbers, dtype=torch.int32, device=device) if numbers else None
    made = (rows, source, offsets)
    done = _run(layout_kernel_plan(), _layout_includes,
                (indices, rows, source, offsets, offsets.view(torch.int32) if scratch is None else scratch, numbers, pairs, indices.size(1), num_experts,
                 current_raw_stream()))
    remember_new(call, *done, made, () if scratch is None else (scratch, ))
    return made


# And back

_combine_includes = ('"moe/combine.hpp"', )

combine_template = """
using namespace yan;
// Templated args from Python JIT call: {TOP_K} rows a token
__return_code = static_cast<int>(launch_moe_combine<{TOP_K}>(reinterpret_cast<const __bf16*>(y), rows_of, weighted ? weights : nullptr,
                                                             reinterpret_cast<__bf16*>(out), tokens, columns, rows, stream));
"""
combine_arg_defs = (('y', torch.bfloat16), ('rows_of', torch.int), ('weights', torch.float), ('out', torch.bfloat16), ('weighted', int), ('tokens', int),
                    ('columns', int), ('rows', int), ('stream', torch.cuda.Stream))

combine_backward_template = """
using namespace yan;
// Templated args from Python JIT call: {TOP_K} rows a token
__return_code = static_cast<int>(launch_moe_combine_backward<{TOP_K}>(
    reinterpret_cast<const __bf16*>(grad_out), reinterpret_cast<const __bf16*>(y), rows_of, weighted ? weights : nullptr, source,
    reinterpret_cast<__bf16*>(grad_y), weighted ? grad_weights : nullptr, tokens, columns, rows, stream));
"""
combine_backward_arg_defs = (('grad_out', torch.bfloat16), ('y', torch.bfloat16), ('rows_of', torch.int), ('weights', torch.float), ('source', torch.int),
                             ('grad_y', torch.bfloat16), ('grad_weights', torch.float), ('weighted', int), ('tokens', int), ('columns', int), ('rows', int),
                             ('stream', torch.cuda.Stream))


@functools.lru_cache(maxsize=None)
def combine_kernel_plan(top_k: int, backward: bool = False):
    """(name, keys, arg_defs, template) of the combine kernel; needs no GPU."""
    keys = FrozenKeys({'TOP_K': top_k})
    if backward:
        return 'moe_combine_backward', keys, combine_backward_arg_defs, combine_backward_template
    return 'moe_combine', keys, combine_arg_defs, combine_template


def _check_combine(y, rows, weights, out):
    assert y.dim() == 2 and y.dtype == torch.bfloat16 and y.is_contiguous() and y.size(1) % 8 == 0
    assert rows.dim() == 2 and rows.dtype == torch.int32 and rows.is_contiguous() and 1 <= rows.size(1) <= MAX_TOP_K
    assert out.shape == (rows.size(0), y.size(1)) and out.dtype == torch.bfloat16 and out.is_contiguous()
    assert y.size(0) < 1 << 31 and rows.size(0) <= MAX_TOKENS
    if weights is not None:
        assert weights.shape == rows.shape and weights.dtype == torch.float32 and weights.is_contiguous()
    assert y.data_ptr() % 16 == 0 and out.data_ptr() % 16 == 0, 'rows start at multiples of 16 bytes'


def moe_combine(y: torch.Tensor, rows: torch.Tensor, weights: Optional[torch.Tensor], out: torch.Tensor) -> None:
    """
    `out[t] = sum_i weights[t, i] * y[rows[t, i]]`: the experts' outputs back to their tokens, summed in fp32.

    y: bf16 `[m, n]`, contiguous, n % 8 == 0 (the masked layout's `[num_experts, m_max, n]` viewed as `[num_experts * m_max, n]`)
    rows: int32 `[tokens, top_k]`, as the dispatch returns them; a row outside of y adds nothing
    weights: fp32 `[tokens, top_k]`, or None for 1 (the gradient of what was dispatched)
    out: bf16 `[tokens, n]`, written in place
    """
    call = (COMBINE, y, rows, weights, out)
    if repeat_call(*call):
        return
    _check_combine(y, rows, weights, out)
    assert_on_current_device(y, rows, weights, out)
    tokens, columns = out.shape
    if tokens == 0 or columns == 0:
        return
    nothing = torch.empty(1, dtype=torch.float32, device=y.device)          # stands for what is not there
    done = _run(combine_kernel_plan(rows.size(1)), _combine_includes,
                (y, rows, nothing if weights is None else weights, out, int(weights is not None), tokens, columns, y.size(0), current_raw_stream()))
    remember_new(call, *done)


def moe_combine_backward(grad_out: torch.Tensor, y: torch.Tensor, rows: torch.Tensor, weights: Optional[torch.Tensor],
                         source: torch.Tensor) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """
    The gradients of `moe_combine`: grad_y bf16 `[m, n]`, zero in rows that no pair has, and grad_weights fp32 `[tokens, top_k]` (None without weights).

    grad_out: bf16 `[tokens, n]`; y, rows, weights: as given to `moe_combine`, no row twice; source: int32 `[m]`, negative for the rows that no
    pair has, as `moe_dispatch_to_fp8_contiguous` returns it
    """
    call = (COMBINE_BACKWARD, grad_out, y, rows, weights, source)
    made = repeat_new(*call)
    if made is not None:
        return made if weights is not None else (made[0], None)
    _check_combine(y, rows, weights, grad_out)
    assert source.shape == (y.size(0), ) and source.dtype == torch.int32 and source.is_contiguous()
    assert_on_current_device(grad_out, y, rows, weights, source)
    tokens, columns = grad_out.shape
    grad_y = torch.empty_like(y)
    grad_weights = None if weights is None else torch.empty_like(weights)
    nothing = torch.empty(1, dtype=torch.float32, device=y.device)          # stands for what is not there
    done = _run(combine_kernel_plan(rows.size(1), True), _combine_includes,
                (grad_out, y, rows, nothing if weights is None else weights, source, grad_y, nothing if weights is None else grad_weights,
                 int(weights is not None), tokens, columns, y.size(0), current_raw_stream()))
    remember_new(call, *done, (grad_y, ) if weights is None else (grad_y, grad_weights))
    return grad_y, grad_weights
