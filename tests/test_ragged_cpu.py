"""The norm, the ragged layout and the ragged products without a GPU: what they refuse, the rules that size their kernels, and what is built of them."""
import ctypes
import os
import random
import re
import subprocess

import pytest
import torch

import yan_amd as yan
from yan_amd.jit import build, cpp_format, generate
from yan_amd.jit.compiler import get_compile_flags, get_hipcc_compiler, get_jit_include_dir
from yan_amd.jit_kernels import moe, norm, ragged

BF16 = torch.bfloat16
NT, NN, TN = yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged, yan.m_grouped_gemm_bf16_bf16_bf16_nn_ragged, yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged


def _refused(fn, *args, **kwargs):
    with pytest.raises(AssertionError):
        fn(*args, **kwargs)


def test_norm_refuses():
    x, w = torch.zeros(4, 256), torch.ones(256)
    fp8 = yan.rms_norm_to_fp8
    _refused(fp8, x.half(), w)
    _refused(fp8, x.t().contiguous().t(), w)
    _refused(fp8, x[None], w)
    _refused(fp8, x[:, :192].contiguous(), w[:192])                     # no whole blocks of 128
    _refused(fp8, x, w[:128])
    _refused(fp8, x, w.half())
    _refused(fp8, x, w[None])
    _refused(fp8, x, w, -1e-6)
    _refused(fp8, x, w, float('nan'))
    _refused(fp8, x, w, 1e-6, x[:3])
    _refused(fp8, x, w, 1e-6, x.half())
    _refused(fp8, x, w, 1e-6, torch.zeros(256, 4).t())
    _refused(fp8, x, w, 1e-6, None, False, x)                           # 16 bits are bf16
    _refused(fp8, x, w, 1e-6, None, False, x.bfloat16()[:3])
    _refused(fp8, torch.zeros(1025)[1:].view(4, 256), w)                # not at a multiple of 16 bytes
    _refused(fp8, torch.zeros(1, norm.MAX_COLUMNS + 128), torch.ones(norm.MAX_COLUMNS + 128))
    _refused(fp8, torch.zeros(4, 0), torch.zeros(0))
    _refused(yan.rms_norm, x, w, None)
    _refused(yan.rms_norm, x, w, x)
    _refused(yan.rms_norm, x[:, :100].contiguous(), w[:100], x[:, :100].bfloat16().contiguous())
    back, r = yan.rms_norm_backward, torch.ones(4)
    _refused(back, x, x[:3], w, r)
    _refused(back, x, x, w, r[:3])
    _refused(back, x, x, w, r.double())
    _refused(back, x, x, w, r, torch.zeros(255))
    _refused(back, x, x, w, r, torch.zeros(256, dtype=BF16))
    _refused(back, x, x, w, r, None, x.bfloat16())                      # of grad_out's type
    _refused(back, x, x, w, r, None, x[:3])
    _refused(back, x.half(), x, w, r)


def test_norm_refuses_its_residual_for_its_output():
    x, residual, w = torch.zeros(4, 256, dtype=BF16), torch.zeros(4, 256, dtype=BF16), torch.ones(256)
    with pytest.raises(AssertionError, match='a place of their own'):
        yan.rms_norm(x, w, residual, 1e-6, residual)
    with pytest.raises(AssertionError, match='a place of their own'):
        yan.rms_norm_to_fp8(x, w, 1e-6, residual, False, residual)


def test_layout_refuses():
    i = torch.zeros(4, 2, dtype=torch.int32)
    _refused(yan.moe_ragged_layout, i.long(), 4)
    _refused(yan.moe_ragged_layout, i[0], 4)
    _refused(yan.moe_ragged_layout, i.t(), 4)
    _refused(yan.moe_ragged_layout, i, 0)
    _refused(yan.moe_ragged_layout, i, 1025)
    _refused(yan.moe_ragged_layout, torch.zeros(4, 17, dtype=torch.int32), 4)
    _refused(yan.moe_ragged_layout, torch.empty(moe.MAX_PAIRS + 1, 1, dtype=torch.int32, device='meta'), 4)


def test_ragged_products_refuse():
    lhs, rhs, out, offsets = torch.zeros(6, 16, dtype=BF16), torch.zeros(2, 24, 16, dtype=BF16), torch.zeros(6, 24, dtype=BF16), torch.zeros(3, dtype=torch.int32)
    source = torch.zeros(6, dtype=torch.int32)
    _refused(NT, lhs.half(), rhs, out, offsets)
    _refused(NT, lhs, rhs.half(), out, offsets)
    _refused(NT, lhs, rhs, out.float(), offsets)
    _refused(yan.m_grouped_gemm_fp16_fp16_fp16_nt_ragged, lhs, rhs, out, offsets)
    _refused(NT, lhs[:5], rhs, out, offsets)
    _refused(NT, lhs, rhs, out[:, :16].contiguous(), offsets)
    _refused(NT, lhs, rhs[:, :, :8].contiguous(), out, offsets)
    _refused(NT, lhs.t().contiguous().t(), rhs, out, offsets)
    _refused(NT, lhs, rhs.transpose(1, 2).contiguous().transpose(1, 2), out, offsets)
    _refused(NT, lhs, rhs[0], out, offsets)
    _refused(NT, lhs, rhs[:0], out, offsets[:1])
    _refused(NT, lhs, rhs, out, offsets[:2])
    _refused(NT, lhs, rhs, out, offsets.long())
    _refused(NT, lhs, rhs, out, torch.zeros(6, dtype=torch.int32)[::2])
    _refused(NT, lhs, torch.zeros(1025, 24, 16, dtype=BF16), out, torch.zeros(1026, dtype=torch.int32))
    _refused(NT, lhs[:, :12].contiguous(), rhs[:, :, :12].contiguous(), out, offsets)               # k % 8
    _refused(NT, lhs, rhs[:, :20].contiguous(), out[:, :20].contiguous(), offsets)                  # n % 8
    _refused(NT, torch.zeros(97, dtype=BF16)[1:].view(6, 16), rhs, out, offsets)                    # not at a multiple of 16 bytes
    _refused(NT, lhs, rhs, out, offsets, source[:5])
    _refused(NT, lhs, rhs, out, offsets, source.long())
    _refused(NT, lhs[:0], rhs, out, offsets, source)                                                # rows to gather, and none there
    _refused(NN, lhs, rhs, out, offsets)                                                            # its weights are [k, n]
    _refused(NN, lhs, rhs.transpose(1, 2), out, offsets)
    grad, x, dw = torch.zeros(6, 24, dtype=BF16), torch.zeros(6, 16, dtype=BF16), torch.zeros(2, 24, 16)
    _refused(TN, grad, x, dw.bfloat16(), offsets)
    _refused(TN, grad.half(), x, dw, offsets)
    _refused(TN, grad, x, dw.transpose(1, 2), offsets)
    _refused(TN, grad[:5], x, dw, offsets)
    _refused(TN, grad, x, dw[0], offsets)
    _refused(TN, grad, x, dw, offsets[:2])
    _refused(TN, grad, x, dw, offsets, False, source[:5])
    _refused(TN, grad, x[:0], dw, offsets, False, source)
    _refused(TN, grad[:, :20].contiguous(), x, dw[:, :20].contiguous(), offsets)
    meta = lambda *shape, dtype=BF16: torch.empty(shape, dtype=dtype, device='meta')
    # gathered operands of 2 GiB, more rows than a launch counts
    _refused(NT, meta(1 << 26, 16), meta(2, 24, 16), meta(6, 24), meta(3, dtype=torch.int32), meta(6, dtype=torch.int32))
    _refused(NT, meta(1 << 29, 16), meta(2, 24, 16), meta(1 << 29, 24), meta(3, dtype=torch.int32))


def test_norm_kernels_hold_every_row():
    for rows in (1, 1024, 1025, 100000):
        for k in range(8, norm.MAX_COLUMNS + 1, 8):
            lanes, runs = norm.norm_lanes(rows, k)
            assert lanes * runs * 8 >= k and lanes in (16, 64, 256, 1024) and runs in (1, 2, 4, 8)
            lanes, runs = norm.norm_backward_lanes(k)
            assert lanes * runs * 8 >= k and lanes in (16, 64, 256, 1024) and runs in (1, 2, 4) and lanes * runs <= 2048
            assert 1 <= norm.norm_backward_workgroups(rows, k) <= 512


def test_plans_generate():
    plans = [(norm.includes, norm.norm_kernel_plan(BF16, torch.float32, BF16, 256, 4, True, True, True)),
             (norm.includes, norm.norm_backward_kernel_plan(BF16, BF16, torch.float32, 64, 2, False, True)), (moe._layout_includes, moe.layout_kernel_plan())]
    plans += [(ragged.includes, ragged.grouped16_kernel_plan(dtype, mode, gather)) for dtype in (BF16, torch.half) for mode, gather in (('NT', True), ('NN', False), ('TN', True))]
    for includes, (name, keys, arg_defs, template) in plans:
        code = generate(includes, arg_defs, cpp_format(template, dict(keys)))
        assert 'launch_' in code and not any('{' + k + '}' in code for k in keys) and len(arg_defs) <= 20        # what a native repeat call passes


def _asm(tmp_path, includes, plan):
    _, keys, arg_defs, template = plan
    src, asm = tmp_path / 'kernel.cu', tmp_path / 'kernel.s'
    src.write_text(generate(includes, arg_defs, cpp_format(template, dict(keys))))
    flags = [f for f in get_compile_flags() if f not in ('-shared', '-fPIC')]
    subprocess.check_call([get_hipcc_compiler()[0], '-x', 'hip', '--cuda-device-only', '-S', *flags, f'-I{get_jit_include_dir()}', str(src), '-o', str(asm)])
    return asm.read_text()


@pytest.mark.parametrize('mode,gather', [('NT', True), ('NN', False), ('TN', True)])
def test_generated_code_of_the_ragged_products(tmp_path, mode, gather):
    """No store of 16 bytes with part of its offset in a scalar register, whose data may be overwritten in front of it; no wait for all copies, no detour by memory and no copy
    taken lane by lane among the MFMAs of the large tiles."""
    text = _asm(tmp_path, ragged.includes, ragged.grouped16_kernel_plan(BF16, mode, gather))
    lines = [line.split(';')[0].strip() for line in text.split('\n')]
    stores = [line for line in lines if line.startswith('buffer_store_dwordx4')]
    assert len(stores) >= 4 and all(re.match(r'buffer_store_dwordx4 v\[\d+:\d+\], v\d+, s\[\d+:\d+\], 0 ', line) for line in stores), stores[:3]
    tall = text[text.index('grouped16_tall_kernel'):]
    tall = tall[:tall.index('.Lfunc_end')]
    loops = [block for block in re.split(r'\n(?=\.LBB)', tall) if block.count('v_mfma') >= 30]
    assert len(loops) >= 4
    for block in loops:
        between = block[block.index('v_mfma'):block.rindex('v_mfma')]
        assert 'scratch_' not in between and 'vmcnt(0)' not in between and 'v_readfirstlane' not in between


@pytest.mark.parametrize('h,k', [(BF16, 8192), (BF16, 16384), (torch.float32, 16384)])
def test_norm_gradient_stays_in_registers(tmp_path, h, k):
    text = _asm(tmp_path, norm.includes, norm.norm_backward_kernel_plan(BF16, h, BF16, *norm.norm_backward_lanes(k), True, True))
    assert 'rms_norm_backward_kernel' in text and 'scratch_' not in text and not re.search(r'private_segment_fixed_size: *[1-9]', text)


@pytest.mark.parametrize('what', ['products', 'norm', 'layout'])
def test_kernels_are_whole(what):
    """Every kernel that a library launches is in it: the libraries load with all of their symbols."""
    plans = {'products': [(ragged.includes, ragged.grouped16_kernel_plan(BF16, mode, gather)) for mode, gather in (('NT', False), ('NT', True), ('NN', False), ('TN', False), ('TN', True))],
             'norm': [(norm.includes, norm.norm_kernel_plan(BF16, BF16, BF16, 1024, 1, True, True, False)), (norm.includes, norm.norm_backward_kernel_plan(BF16, BF16, BF16, 256, 4, True, True))],
             'layout': [(moe._layout_includes, moe.layout_kernel_plan())]}[what]
    for includes, (name, keys, arg_defs, template) in plans:
        runtime = build(name, arg_defs, generate(includes, arg_defs, cpp_format(template, dict(keys))))
        ctypes.CDLL(os.path.join(runtime.path, 'kernel.so'), mode=os.RTLD_NOW)


def test_every_run_of_rows_has_a_workgroup(tmp_path):
    """As many runs as a launch counts on are enough for any ascending offsets, and the waves' way of looking a run up (64 groups at a time) finds each one once."""
    source, exe = tmp_path / 'runs.cpp', tmp_path / 'runs'
    source.write_text("""
#include "gemm/grouped16.hpp"
#include <cstdio>
int main() {
    int rows, groups, block, runs;
    while (std::scanf("%d %d %d %d", &rows, &groups, &block, &runs) == 4)
        if (runs > yan::most_row_tiles(rows, groups, block)) return 1;
    return 0;
}
""")
    subprocess.check_call([get_hipcc_compiler()[0], '-x', 'hip', '--cuda-host-only', '-std=c++20', '-O1', '-w', f'-I{get_jit_include_dir()}', str(source), '-o', str(exe)])
    rng, cases = random.Random(3), []
    for _ in range(2000):
        groups, block = rng.randint(1, 70), rng.choice([32, 64, 128, 256])
        counts = [rng.choice([0, 1, rng.randint(0, 3 * block), block, block + 1]) for _ in range(groups)]
        cases.append(f'{sum(counts)} {groups} {block} {sum(-(-c // block) for c in counts)}')
    assert subprocess.run([str(exe)], input='\n'.join(cases), text=True).returncode == 0


def test_every_kernel_is_some_calls(tmp_path):
    """The kernel of a product follows from its sizes: each is chosen for some, one that a product does not have for none, and groups without rows or depth have one too."""
    source, exe = tmp_path / 'plan.cpp', tmp_path / 'plan'
    source.write_text("""
#include "gemm/grouped16.hpp"
#include <cstdio>
int main() {
    for (int groups : {1, 4, 16, 64, 1024})
        for (int each : {0, 1, 16, 17, 79, 80, 160, 192, 500, 100000})
            for (int n : {8, 512, 1024, 2048, 7168, (1 << 21) - 8})
                for (int k : {0, 8, 512, 7168}) {
                    const int rows = int(std::min(536870911ll, (long long)each * groups));
                    std::printf("NT %d %d\\n", k == 0, int(yan::grouped16_plan<yan::Grouped::NT>(groups, rows, rows, n, k, 256)));
                    if (k) std::printf("TN %d %d\\n", 0, int(yan::grouped16_plan<yan::Grouped::TN>(groups, rows, k, n, 0, 256)));
                }
}
""")
    subprocess.check_call([get_hipcc_compiler()[0], '-x', 'hip', '--cuda-host-only', '-std=c++20', '-O1', '-w', f'-I{get_jit_include_dir()}', str(source), '-o', str(exe)])
    chosen = {}
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split('\n')[:-1]:
        mode, shallow, kernel = line.split()
        chosen.setdefault(f'{mode} {shallow}', set()).add(int(kernel))
    # kGroupedTall, kGrouped128, kGrouped64, kGrouped32
    assert chosen == {'NT 0': {1, 2, 3, 4}, 'NT 1': {2, 3, 4}, 'TN 0': {1, 2, 3}}


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
        for module in (moe, norm, ragged):
            monkeypatch.setattr(module, 'current_raw_stream', lambda: 0)
            monkeypatch.setattr(module, 'assert_on_current_device', lambda *_: None)
        monkeypatch.setattr(ragged, 'get_num_sms', lambda: 256)

    def tensors(self, arg_defs, call):
        """By name: which of the noted call's tensors each of the launch's is, None for one that the caller did not give. Floats go where floats go and are in no place of their own."""
        call()
        (_, _, _, spec, *_), = self.noted
        self.noted.clear()
        defs = [d for d in arg_defs if d[1] is not float]
        assert len(spec) == len(defs)
        return {name: value if kind == 0 else None for (name, dtype), (kind, value) in zip(defs, spec) if isinstance(dtype, torch.dtype)}


def test_notes_of_a_call_say_which_argument_is_which(monkeypatch):
    notes = _Notes(monkeypatch)
    meta = lambda *shape, dtype=BF16: torch.empty(shape, dtype=dtype, device='meta')
    x, w, residual, out = meta(4, 128), meta(128), meta(4, 128), meta(4, 128)
    defs = norm.norm_kernel_plan(BF16, BF16, BF16, 16, 1, True, True, True)[2]
    made = {'codes': None, 'scales': None, 'inverse_rms': None}
    assert notes.tensors(defs, lambda: yan.rms_norm_to_fp8(x, w, 1e-6, residual, True, out)) == {'x': 0, 'weight': 1, 'residual': 2, 'normed': 3, **made}
    assert notes.tensors(defs, lambda: yan.rms_norm_to_fp8(x, w)) == {'x': 0, 'weight': 1, 'residual': None, 'normed': None, **made}
    assert notes.tensors(defs, lambda: yan.rms_norm(x, w, out)) == {'x': 0, 'weight': 1, 'residual': None, 'normed': 2, **made}
    assert notes.tensors(defs, lambda: yan.rms_norm(x, w, x, 1e-6, residual)) == {'x': 0, 'weight': 1, 'residual': 2, 'normed': 3, **made}
    defs = norm.norm_backward_kernel_plan(BF16, BF16, BF16, 16, 1, True, True)[2]
    r, dw = meta(4, dtype=torch.float32), meta(128, dtype=torch.float32)
    for grad in (x, residual):
        got = notes.tensors(defs, lambda: yan.rms_norm_backward(grad, residual, w, r, dw, grad))
        assert got == {'grad': 0, 'h': 1, 'weight': 2, 'inverse_rms': 3, 'grad_weight': 4, 'grad_residual': 5, 'grad_h': None, 'partial': None}
        got = notes.tensors(defs, lambda: yan.rms_norm_backward(grad, residual, w, r, None, grad))
        assert got == {'grad': 0, 'h': 1, 'weight': 2, 'inverse_rms': 3, 'grad_weight': None, 'grad_residual': 4, 'grad_h': None, 'partial': None}
    picks = meta(4, 2, dtype=torch.int32)
    assert notes.tensors(moe.layout_arg_defs, lambda: yan.moe_ragged_layout(picks, 8)) == {'indices': 0, 'rows': None, 'source': None, 'offsets': None, 'workspace': None}
    lhs, rhs, offsets, source = meta(8, 16), meta(2, 8, 16), meta(3, dtype=torch.int32), meta(8, dtype=torch.int32)
    defs = ragged.grouped16_kernel_plan(BF16, 'NT', True)[2]
    product = meta(8, 8)
    assert notes.tensors(defs, lambda: NT(lhs, rhs, product, offsets, source)) == {'lhs': 0, 'rhs': 1, 'out': 2, 'offsets': 3, 'source': 4}
    assert notes.tensors(defs, lambda: NT(lhs, rhs, product, offsets)) == {'lhs': 0, 'rhs': 1, 'out': 2, 'offsets': 3, 'source': None}
    for left in (lhs, meta(8, 16)):                 # the same tensor on both sides and then two
        assert notes.tensors(defs, lambda: TN(left, lhs, meta(2, 16, 16, dtype=torch.float32), offsets, True, source)) == {'lhs': 0, 'rhs': 1, 'out': 2, 'offsets': 3, 'source': 4}
