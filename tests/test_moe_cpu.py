"""The mixture-of-experts entries and the weight-gradient products without a GPU: what they refuse, and the rules that size their kernels."""
import ctypes
import random
import re

import pytest
import torch

import yan_amd as yan
from yan_amd.jit import cpp_format, generate
from yan_amd.jit_kernels import fp8_cast, moe, wgrad

F8 = torch.float8_e4m3fn


def test_plans_generate_and_are_shared_between_sizes():
    for dtype in (torch.bfloat16, torch.float32):
        for scoring in ('softmax', 'sigmoid'):
            for backward in (False, True):
                plans = {moe.route_kernel_plan(dtype, scoring, experts, backward)[1]['LANES'] * 100 + moe.route_kernel_plan(dtype, scoring, experts, backward)[1]['VALUES']
                         for experts in range(1, 1025)}
                assert len(plans) == 5
        for plan in (moe.dispatch_kernel_plan(dtype), fp8_cast.cast_kernel_plan('per_channel', dtype), moe.route_kernel_plan(dtype, 'softmax', 8)):
            name, keys, arg_defs, template = plan
            code = generate(('"moe/route.hpp"', ), arg_defs, cpp_format(template, dict(keys)))
            assert 'launch_' in code and not any('{' + k + '}' in code for k in keys)
    assert len(wgrad.arg_defs) <= 20 and len(moe.dispatch_kernel_plan(torch.bfloat16)[2]) <= 20      # what a native repeat call passes


def test_lanes_hold_every_number_of_experts():
    for experts in range(1, moe.MAX_EXPERTS + 1):
        lanes, values = moe.route_lanes(experts)
        assert lanes * values >= experts and lanes in (16, 32, 64) and lanes >= moe.MAX_TOP_K
        for tokens in (0, 1, 15, 16, 17, 100, 4096, 1 << 20):
            assert 1 <= moe.route_blocks(tokens, experts) <= 256


def test_contiguous_rows_are_enough_and_no_more_than_that():
    rng = random.Random(5)
    for _ in range(300):
        tokens, top_k, experts = rng.randint(1, 200), rng.randint(1, 8), rng.randint(1, 40)
        most = yan.get_contiguous_layout_rows(tokens, top_k, experts)
        assert most % 128 == 0
        for _ in range(10):
            counts = [0] * experts
            for _ in range(tokens * top_k):
                counts[rng.randrange(experts) if rng.random() < 0.8 else 0] += 1
            assert sum((c + 127) // 128 * 128 for c in counts) <= most
    # every expert but one has one pair, the last one the rest: the bound is reached
    assert yan.get_contiguous_layout_rows(128, 1, 4) == 3 * 128 + 128 and yan.get_contiguous_layout_rows(0, 8, 4) == 0
    assert yan.get_contiguous_layout_rows(1, 1, 256) == 128


def _refused(fn, *args, **kwargs):
    with pytest.raises(AssertionError):
        fn(*args, **kwargs)


def test_route_refuses():
    x = torch.zeros(4, 8)
    _refused(yan.moe_route, x, 9)
    _refused(yan.moe_route, x, 0)
    _refused(yan.moe_route, torch.zeros(4, 64), 17)
    _refused(yan.moe_route, torch.zeros(4, 1025), 2)
    _refused(yan.moe_route, x.half(), 2)
    _refused(yan.moe_route, x, 2, 'tanh')
    _refused(yan.moe_route, torch.zeros(8, 4).t(), 2)
    _refused(yan.moe_route, x[None], 2)
    _refused(yan.moe_route, x, 2, mask=torch.ones(3, dtype=torch.bool))
    _refused(yan.moe_route, x, 2, mask=torch.ones(4, dtype=torch.uint8))
    i, c, w, l = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(4, 2), torch.zeros(())
    _refused(yan.moe_route_backward, x, i.long(), c, w, l)
    _refused(yan.moe_route_backward, x, i[:3], c, w[:3], l)
    _refused(yan.moe_route_backward, x, i, c[:7], w, l)
    _refused(yan.moe_route_backward, x, i, c, w[:, :1], l)
    _refused(yan.moe_route_backward, x, i, c, w, torch.zeros(2))
    _refused(yan.moe_route_backward, x, i, c, w.double(), l)
    _refused(yan.moe_route_backward, x, i, c, w, l, 'tanh')
    _refused(yan.moe_route_backward, x, i[:, 0], c, w, l)


def test_dispatch_refuses():
    x, i = torch.zeros(4, 256), torch.zeros(4, 2, dtype=torch.int32)
    codes, scales = torch.zeros(512, 256, dtype=torch.uint8).view(F8), torch.zeros(512, 2)
    _refused(yan.moe_dispatch_to_fp8_contiguous, x, i, 1025, (codes, scales))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x, i, 0, (codes, scales))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x, i[:3], 4, (codes, scales))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x, i.long(), 4, (codes, scales))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x.half(), i, 4, (codes, scales))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x[:, :200].contiguous(), i, 4, (codes, scales))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x, i, 4, (codes[:500], scales[:500]))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x, i, 4, (codes, scales[:, :1]))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x, i, 4, (codes, scales.double()))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x, torch.zeros(4, 17, dtype=torch.int32), 4, (codes, scales))
    _refused(yan.moe_dispatch_to_fp8_contiguous, x, i, 4, (codes.view(4, 128, 256), scales.view(4, 128, 2)))
    _refused(yan.moe_dispatch_to_fp8_masked, x, i, (codes, scales))
    _refused(yan.moe_dispatch_to_fp8_masked, x, i, (codes.view(4, 128, 256)[:, :100], scales.view(4, 128, 2)[:, :100]))
    _refused(yan.moe_dispatch_to_fp8_masked, x, i, (codes.view(4, 128, 256), scales.view(4, 2, 128)))


def test_combine_refuses():
    y, rows, w, out = torch.zeros(128, 64, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2), torch.zeros(4, 64, dtype=torch.bfloat16)
    source = torch.zeros(128, dtype=torch.int32)
    _refused(yan.moe_combine, y.float(), rows, w, out)
    _refused(yan.moe_combine, y[:, :60].contiguous(), rows, w, out[:, :60].contiguous())
    _refused(yan.moe_combine, y.t(), rows, w, out)
    _refused(yan.moe_combine, y, rows.long(), w, out)
    _refused(yan.moe_combine, y, torch.zeros(4, 17, dtype=torch.int32), None, out)
    _refused(yan.moe_combine, y, rows, w[:3], out)
    _refused(yan.moe_combine, y, rows, w.bfloat16(), out)
    _refused(yan.moe_combine, y, rows, w, out[:3])
    _refused(yan.moe_combine, y, rows, w, out.float())
    _refused(yan.moe_combine, y.view(2, 64, 64), rows, w, out)
    _refused(yan.moe_combine_backward, out, y, rows, w, source[:64])
    _refused(yan.moe_combine_backward, out, y, rows, w, source.long())
    _refused(yan.moe_combine_backward, out[:3], y, rows, w, source)


def test_per_channel_cast_refuses():
    x = torch.zeros(8, 16)
    _refused(yan.per_channel_cast_to_fp8, x[:, :12].contiguous())
    _refused(yan.per_channel_cast_to_fp8, x.t())
    _refused(yan.per_channel_cast_to_fp8, x[None])
    _refused(yan.per_channel_cast_to_fp8, x.half())
    _refused(yan.per_channel_cast_to_fp8, x, torch.zeros(100, dtype=torch.int32))
    _refused(yan.per_channel_cast_to_fp8, x, torch.zeros(128, dtype=torch.int64))
    _refused(yan.per_channel_cast_to_fp8, x, torch.zeros(2, 64, dtype=torch.int32))
    _refused(yan.per_channel_cast_to_fp8, x, torch.zeros(129, dtype=torch.int32)[1:])          # not at a multiple of 16 bytes


def _operand(rows, k):
    codes, scales = torch.zeros(rows, k, dtype=torch.uint8).view(F8), torch.zeros(rows, (k // 128 + 3) // 4 * 4, dtype=torch.uint8)[:, :k // 128]
    return codes, scales


def test_weight_gradients_refuse():
    a, b, out = _operand(16, 640), _operand(8, 640), torch.zeros(16, 8)
    gemm, grouped = yan.gemm_fp8_fp8_fp32_nt, yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous
    _refused(gemm, a, b, out.bfloat16())
    _refused(gemm, a, b, out[:15])
    _refused(gemm, a, b, out[None])
    _refused(gemm, a, _operand(8, 512), out)
    _refused(gemm, a, _operand(6, 640), torch.zeros(16, 6))
    _refused(gemm, (a[0], a[1].float()), b, out)
    _refused(gemm, (a[0], a[1].contiguous()), b, out)                      # rows five bytes apart
    _refused(gemm, (a[0], a[1][:, :4]), b, out)
    _refused(gemm, (a[0][:, :600], a[1]), b, out)
    _refused(gemm, (a[0].view(torch.uint8), a[1]), b, out)
    _refused(gemm, (a[0], torch.zeros(5, 16, dtype=torch.uint8).t()), b, out)
    _refused(gemm, a, b, torch.zeros(8, 16).t())
    offsets = torch.zeros(3, dtype=torch.int32)
    _refused(grouped, a, b, out, offsets)
    _refused(grouped, a, b, torch.zeros(2, 16, 8), offsets[:2])
    _refused(grouped, a, b, torch.zeros(2, 16, 8), offsets.long())
    _refused(grouped, a, b, torch.zeros(0, 16, 8), offsets[:1])


def test_more_tokens_than_a_launch_counts_are_refused():
    most = moe.MAX_TOKENS
    for tokens in (most, most + 1):
        logits, out = torch.empty(tokens, 4, device='meta'), torch.empty(tokens, 8, dtype=torch.bfloat16, device='meta')
        y, rows = torch.empty(4, 8, dtype=torch.bfloat16, device='meta'), torch.empty(tokens, 1, dtype=torch.int32, device='meta')
        if tokens <= most:
            moe._check_route(logits, 2, 'softmax')
        else:
            _refused(moe._check_route, logits, 2, 'softmax')
            _refused(moe._check_combine, y, rows, None, out)


def test_more_pairs_than_row_numbers_hold_are_refused():
    """Rows are numbers of 32 bits, with every expert's rounded up, and so are the places of a chunk's pairs behind the last token."""
    for tokens, top_k, experts in ((143165576, 15, 16), (143165576, 15, 1), ((1 << 27) - 1, 16, 4), ((1 << 31) - 1, 1, 64)):
        x, indices = torch.empty(tokens, 128, dtype=torch.bfloat16, device='meta'), torch.empty(tokens, top_k, dtype=torch.int32, device='meta')
        codes, scales = torch.empty(256, 128, dtype=F8, device='meta'), torch.empty(256, 1, device='meta')
        _refused(moe._check_dispatch, x, indices, codes, scales, experts)
    most = moe.MAX_PAIRS
    assert most + 127 * moe.MAX_EXPERTS < 1 << 31 and most + moe.TOKENS_PER_BLOCK * moe.MAX_TOP_K < 1 << 31
    for pairs, taken in ((most, True), (most + 1, False)):
        x, indices = torch.empty(pairs, 128, dtype=torch.bfloat16, device='meta'), torch.empty(pairs, 1, dtype=torch.int32, device='meta')
        if taken:
            moe._check_dispatch(x, indices, codes, scales, moe.MAX_EXPERTS)
        else:
            _refused(moe._check_dispatch, x, indices, codes, scales, moe.MAX_EXPERTS)


def _stores_of_16_bytes(tmp_path, code):
    import subprocess
    from yan_amd.jit.compiler import get_hipcc_compiler, get_jit_include_dir, get_offload_arch
    src, asm = tmp_path / 'kernel.cu', tmp_path / 'kernel.s'
    src.write_text(code)
    subprocess.check_call([get_hipcc_compiler()[0], '-x', 'hip', '--cuda-device-only', '-S', '-std=c++20', '-O3', f'--offload-arch={get_offload_arch()}',
                           '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops', f'-I{get_jit_include_dir()}', str(src), '-o', str(asm)])
    lines = [line.split(';')[0].strip() for line in asm.read_text().split('\n')]
    return [line for line in lines if line.startswith('buffer_store_dwordx4')]


@pytest.mark.parametrize('which', ['weight gradients', 'bf16 split-K', 'FP8 split-K'])
def test_no_store_of_16_bytes_has_a_scalar_offset(tmp_path, which):
    """Such a store may read its data after the next vector instruction has overwritten it, and the compiler leaves it without a wait."""
    from yan_amd.jit_kernels import bf16_gemm, gemm
    if which == 'weight gradients':
        _, keys, arg_defs, template = wgrad.wgrad_kernel_plan()
        includes = wgrad.includes
    elif which == 'bf16 split-K':
        _, keys, arg_defs = bf16_gemm.dense_split_k_plan(256, 5120, 5120, torch.bfloat16, 256)
        includes, template = bf16_gemm.includes, bf16_gemm.split_k_template
    else:
        _, keys, arg_defs, template = gemm.fp8_split_k_plan(64, 4096, 7168, 256)
        includes = gemm.includes
    stores = _stores_of_16_bytes(tmp_path, generate(includes, arg_defs, cpp_format(template, dict(keys))))
    # vector data, vector offset, descriptor, scalar offset with the modifiers behind it
    # (the smallest, 64 x 64 on 8 waves: two vectors of partial sums a lane, one of outputs in either of two policies)
    assert len(stores) >= 4 and all(re.match(r'buffer_store_dwordx4 v\[\d+:\d+\], v\d+, s\[\d+:\d+\], 0 ', line) for line in stores), stores[:3]


class _Notes:
    """Stands in for the device and for the native module: launches report success, and what is noted of them is kept."""

    def __init__(self, monkeypatch):
        from yan_amd.jit.runtime import Runtime
        from yan_amd.jit_kernels import host_calls, utils
        self.noted = []
        for name in ('YAN_SPLIT_K', 'YAN_TUNE_TILES'):
            monkeypatch.delenv(name, raising=False)
        monkeypatch.setattr(host_calls, '_host_calls', type('Module', (), {'remember': staticmethod(lambda *note: self.noted.append(note))}))
        monkeypatch.setattr(host_calls, 'repeat_new', lambda *_: None)
        monkeypatch.setattr(utils, '_num_sms', 256)
        monkeypatch.setattr(Runtime, 'is_path_valid', staticmethod(lambda path: True))
        monkeypatch.setattr(Runtime, '__call__', lambda self, *args: 0)

        def compile_and_tune(name, arg_defs, **_):
            runtime = Runtime(name)
            runtime._launch, runtime.args = ctypes.CFUNCTYPE(None)(lambda: None), arg_defs
            return runtime
        monkeypatch.setattr(moe.jit_tuner, 'compile_and_tune', compile_and_tune)
        for module in (moe, wgrad, fp8_cast):
            monkeypatch.setattr(module, 'current_raw_stream', lambda: 0)
            monkeypatch.setattr(module, 'assert_on_current_device', lambda *_: None)
        monkeypatch.setattr(wgrad, 'get_num_sms', lambda: 256)
        for module in (moe, wgrad):
            monkeypatch.setattr(module, 'split_k_workspace', lambda device, stream: (torch.empty(8, dtype=torch.uint8, device='meta'), None))

    def tensors(self, arg_defs, call):
        """By name: which of the noted call's tensors each of the launch's is, None for one that the caller did not give."""
        call()
        (_, _, _, spec, *_), = self.noted
        self.noted.clear()
        assert len(spec) == len(arg_defs)
        return {name: value if kind == 0 else None for (name, dtype), (kind, value) in zip(arg_defs, spec) if isinstance(dtype, torch.dtype)}


def test_notes_of_a_call_say_which_argument_is_which_also_where_two_are_the_same(monkeypatch):
    """A later call of the same sizes takes its addresses by place: it may have two tensors where the noted one had the same twice."""
    notes = _Notes(monkeypatch)
    meta = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device='meta')
    a, b = [(meta(64, 512, dtype=F8), meta(64, 4, dtype=torch.uint8)) for _ in range(2)]
    out, offsets = meta(64, 64), meta(3, dtype=torch.int32)
    want = {'lhs': 0, 'lhs_scales': 1, 'rhs': 2, 'rhs_scales': 3, 'out': 4, 'offsets': None, 'workspace': None}
    for lhs, rhs in ((a, b), (a, a), (a, (b[0], a[1])), (a, (a[0], b[1]))):
        assert notes.tensors(wgrad.arg_defs, lambda: yan.gemm_fp8_fp8_fp32_nt(lhs, rhs, out)) == want
        assert notes.tensors(wgrad.arg_defs, lambda: yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(lhs, rhs, meta(2, 64, 64), offsets)) == {**want, 'offsets': 5}
    y, d, rows, w, source = meta(4, 64, dtype=torch.bfloat16), meta(4, 64, dtype=torch.bfloat16), meta(4, 2, dtype=torch.int32), meta(4, 2), meta(4, dtype=torch.int32)
    for grad_out in (d, y):
        got = notes.tensors(moe.combine_backward_arg_defs, lambda: yan.moe_combine_backward(grad_out, y, rows, w, source))
        assert got == {'grad_out': 0, 'y': 1, 'rows_of': 2, 'weights': 3, 'source': 4, 'grad_y': None, 'grad_weights': None}
        got = notes.tensors(moe.combine_backward_arg_defs, lambda: yan.moe_combine_backward(grad_out, y, rows, None, source))
        assert got == {'grad_out': 0, 'y': 1, 'rows_of': 2, 'weights': None, 'source': 3, 'grad_y': None, 'grad_weights': None}
    for weights, after in ((w, 3), (None, 2)):
        got = notes.tensors(moe.combine_arg_defs, lambda: yan.moe_combine(y, rows, weights, d))
        assert got['y'] == 0 and got['rows_of'] == 1 and sorted(v for v in got.values() if v is not None) == list(range(after + 1))
        assert (got['weights'] is None) == (weights is None) and got['weights'] != got['out']
    logits, indices, counts, loss = meta(4, 2), meta(4, 2, dtype=torch.int32), meta(2, dtype=torch.int32), meta()
    defs = moe.route_kernel_plan(torch.float32, 'softmax', 2, True)[2]
    for grad_weights in (w, logits):
        got = notes.tensors(defs, lambda: yan.moe_route_backward(logits, indices, counts, grad_weights, loss))
        assert got == {'logits': 0, 'indices': 1, 'counts': 2, 'grad_weights': 3, 'grad_loss': 4, 'grad_logits': None}
    got = notes.tensors(defs, lambda: yan.moe_route_backward(logits, indices, counts, None, loss))
    assert got == {'logits': 0, 'indices': 1, 'counts': 2, 'grad_weights': None, 'grad_loss': 3, 'grad_logits': None}
    defs = moe.route_kernel_plan(torch.float32, 'softmax', 2)[2]
    for mask in (None, meta(4, dtype=torch.bool)):
        got = notes.tensors(defs, lambda: yan.moe_route(logits, 1, mask=mask))
        assert got['logits'] == 0 and got['mask'] == (None if mask is None else 1)
    x, codes, scales = meta(4, 128, dtype=torch.bfloat16), meta(128, 128, dtype=F8), meta(128, 1)
    got = notes.tensors(moe.dispatch_kernel_plan(x.dtype)[2], lambda: yan.moe_dispatch_to_fp8_contiguous(x, indices, 2, (codes, scales)))
    assert [got[name] for name in ('x', 'indices', 'codes', 'scales', 'rows_of')] == [0, 1, 2, 3, None]
    got = notes.tensors(moe.dispatch_kernel_plan(x.dtype)[2], lambda: yan.moe_dispatch_to_fp8_masked(x, indices, (codes.view(2, 64, 128), scales.view(2, 64, 1))))
    assert [got[name] for name in ('x', 'indices', 'codes', 'scales', 'rows_of')] == [0, 1, 2, 3, None]
    for picked in (None, meta(128, dtype=torch.int32)):
        got = notes.tensors(fp8_cast.per_channel_arg_defs(x.dtype), lambda: yan.per_channel_cast_to_fp8(x, picked))
        assert got == {'x': 0, 'source': None if picked is None else 1, 'q': None, 'scales': None}


def test_weight_gradient_kernels_are_whole():
    """Every kernel that a library of theirs launches is in it: the library loads with all of its symbols."""
    import os
    from yan_amd.jit import build
    name, keys, arg_defs, template = wgrad.wgrad_kernel_plan()
    runtime = build(name, arg_defs, generate(wgrad.includes, arg_defs, cpp_format(template, dict(keys))))
    ctypes.CDLL(os.path.join(runtime.path, 'kernel.so'), mode=os.RTLD_NOW)


def test_no_copy_of_a_weight_gradient_is_out_of_range_for_every_lane(tmp_path):
    """The LDS that the copies go to is used again: each one has a row to wait for, whatever the operand's number of rows."""
    import subprocess
    from yan_amd.jit.compiler import get_hipcc_compiler, get_jit_include_dir
    source, exe = tmp_path / 'rows.cpp', tmp_path / 'rows'
    source.write_text("""
#include "gemm/fp8_wgrad.hpp"
template <int ROWS>
int check() {
    using Stager = yan::WgradStager<ROWS, 4>;
    for (int rows = 1; rows <= ROWS; ++rows)
        for (int group = 0; group < Stager::PASSES * 4; ++group) {
            const int from = Stager::source_group(group, rows);
            if (from < 0 || from * 8 >= rows || (group * 8 < rows && from != group)) return 1;
        }
    return Stager::PASSES * 32 != ROWS;
}
int main() { return check<64>() + check<128>() + check<256>(); }
""")
    subprocess.check_call([get_hipcc_compiler()[0], '-x', 'hip', '--cuda-host-only', '-std=c++20', '-O1', '-w', f'-I{get_jit_include_dir()}', str(source),
                           '-o', str(exe)])
    assert subprocess.run([str(exe)]).returncode == 0
