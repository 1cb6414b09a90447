"""Edges of the norm, the ragged layout and the ragged products that a host can look at: ranges of descriptors, numbers near the ends of their types, refusals."""
import itertools
import random
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

import yan_amd as yan
from yan_amd.jit import cpp_format, generate
from yan_amd.jit.compiler import get_compile_flags, get_hipcc_compiler, get_jit_include_dir
from yan_amd.jit_kernels import moe, norm, ragged


def _host(tmp_path, body, lines=''):
    """What a program of the kernels' headers, built for the host, says to `lines`."""
    source, exe = tmp_path / 'host.cpp', tmp_path / 'host'
    source.write_text(body)
    subprocess.check_call([get_hipcc_compiler()[0], '-x', 'hip', '--cuda-host-only', '-std=c++20', '-O1', '-w', f'-I{get_jit_include_dir()}', str(source), '-o', str(exe)])
    return subprocess.run([str(exe)], input=lines, capture_output=True, text=True, check=True).stdout.split('\n')[:-1]


# rows, columns of gathered operands of less than 2 GiB by less than a row or by less than the descriptors' bias
NEARLY_2_GIB = [(508400, 2112), (2097151, 512), (1048575, 1024), ((1 << 27) - 1, 8), (2064888, 520), (699050, 1536), (262143, 4096)]


def test_large_tiles_reach_the_end_of_gathered_operands(tmp_path):
    """The descriptors of the large tiles start early: what they reach ends where the operand does, for every size that is accepted."""
    out = _host(tmp_path, """
#include "gemm/grouped16.hpp"
#include <cstdio>
int main() {
    long long bytes;
    while (std::scanf("%lld", &bytes) == 1) std::printf("%u\\n", yan::biased_reach(bytes));
    std::printf("%u\\n", yan::kCopyBias);
}
""", '\n'.join(str(2 * rows * columns) for rows, columns in NEARLY_2_GIB + [(1, 8), (1 << 20, 256)]))
    bias = int(out[-1])
    assert bias > 0
    for (rows, columns), reached in zip(NEARLY_2_GIB + [(1, 8), (1 << 20, 256)], out):
        assert 2 * rows * columns < 1 << 31 and int(reached) == 2 * rows * columns + bias
        # the farthest byte that a copy asks for, behind a k-tile of the last row, is a number of 32 bits
        assert 2 * rows * columns + bias + 128 < 1 << 32


def test_copies_of_turned_weights_have_rows(tmp_path):
    """Large tiles copy whole k-tiles of [k, n] weights unless the operand ends inside: two rows an instruction, one of which at least has to exist, for any depth and group."""
    cases = [(groups, k) for groups in (1, 2, 3, 7, 8, 9, 64, 1024) for k in [*range(8, 200, 8), 1544, (1 << 21) - 8]]
    out = _host(tmp_path, """
#include "gemm/grouped16.hpp"
#include <cstdio>
int main() {
    int left, k;
    while (std::scanf("%d %d", &left, &k) == 2) std::printf("%d\\n", int(yan::weights_end_inside(left, k)));
}
""", '\n'.join(f'{groups - group} {k}' for groups, k in cases for group in range(groups)))
    answers = iter(out)
    for groups, k in cases:
        whole = -(-k // 64) * 64
        for group in range(groups):
            inside = next(answers) == '1'
            assert inside == (group * k + whole > groups * k), (groups, group, k)
            # (otherwise the last k-tile's rows behind the contraction stand for its last row)
            if not inside:
                assert all(group * k + row < groups * k for row in range(whole - 64, whole)), (groups, group, k)


def test_rows_of_the_norm_up_to_31_bits(tmp_path):
    """Every row is some group of lanes' and a group without one has the last, up to as many rows as there are numbers for."""
    out = _host(tmp_path, """
#include "norm/rms_norm.hpp"
#include <cstdio>
template <int ROWS> int check(int rows) {
    const int blocks = yan::norm_blocks<ROWS>(rows);
    if (blocks != int(((long long)rows + ROWS - 1) / ROWS)) return 1;
    for (int b : {0, blocks / 2, blocks - 1})
        for (int g = 0; g < ROWS; ++g) {
            const long long row = (long long)b * ROWS + g;
            if (yan::norm_row_exists<ROWS>(b, g, rows) != (row < rows) || yan::norm_row<ROWS>(b, g, rows) != int(row < rows ? row : rows - 1)) return 2;
        }
    return 0;
}
int main() {
    int rows;
    while (std::scanf("%d", &rows) == 1) std::printf("%d %d %d\\n", check<1>(rows), check<4>(rows), check<16>(rows));
}
""", '\n'.join(str(r) for r in [*range(1, 40), 1 << 28, (1 << 31) - 17, (1 << 31) - 16, (1 << 31) - 15, (1 << 31) - 4, (1 << 31) - 2, (1 << 31) - 1]))
    assert len(out) == 46 and all(line == '0 0 0' for line in out)


def test_norm_refuses_any_part_of_its_residual_for_its_output():
    """Views of the residual, and tensors that only share some bytes with it, are no place for the normed rows: these would take the sums' place, which the next layer and the gradient read."""
    memory, w = torch.zeros(12, 256, dtype=torch.bfloat16), torch.ones(256)
    residual, x = memory[4:8], torch.zeros(4, 256, dtype=torch.bfloat16)
    wide = torch.zeros(4, 256)                      # fp32: its first and its last half as 16 bits
    inside = [(residual, out) for out in (residual.view(4, 256), residual[:], memory[4:8], memory[1:5], memory[7:11])]
    inside += [(wide, wide.view(torch.bfloat16).view(8, 256)[at:at + 4]) for at in (0, 2, 4)]
    for r, out in inside:
        with pytest.raises(AssertionError, match='a place of their own'):
            yan.rms_norm(x, w, out, 1e-6, r)
        with pytest.raises(AssertionError, match='a place of their own'):
            yan.rms_norm_to_fp8(x, w, 1e-6, r, False, out)
    # neighbours are places of their own, and so are rows of none: refused for not being on a device at most
    for r, out in ((residual, memory[:4]), (residual, memory[8:]), (memory[4:4], memory[4:4])):
        with pytest.raises((AssertionError, RuntimeError)) as refusal:
            yan.rms_norm(x[:r.size(0)], w, out, 1e-6, r)
        assert 'a place of their own' not in str(refusal.value)


def test_types_of_the_ragged_entries_are_part_of_what_calls_are_found_by(monkeypatch):
    """A call that was served once is found by what it was given: the bf16 and the fp16 entry with the same tensors are two calls."""
    asked = []
    monkeypatch.setattr(ragged, 'repeat_call', lambda *call: asked.append(call) or True)
    lhs, weights, out, offsets = torch.zeros(6, 16, dtype=torch.bfloat16), torch.zeros(2, 16, 16, dtype=torch.bfloat16), torch.zeros(6, 16, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    for one, other in ((yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged, yan.m_grouped_gemm_fp16_fp16_fp16_nt_ragged),
                       (yan.m_grouped_gemm_bf16_bf16_bf16_nn_ragged, yan.m_grouped_gemm_fp16_fp16_fp16_nn_ragged),
                       (yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged, yan.k_grouped_gemm_fp16_fp16_fp32_tn_ragged)):
        one(lhs, weights, out, offsets)
        other(lhs, weights, out, offsets)
        first, second = ([part for part in call if not isinstance(part, torch.Tensor)] for call in asked[-2:])
        assert first != second


def test_norm_launches_hold_their_rows(tmp_path):
    """A launch's workgroups, a whole number for every XCD, have less than 2^32 threads and the rows that it is given."""
    out = _host(tmp_path, """
#include "norm/rms_norm.hpp"
#include <cstdio>
int main() {
    for (int lanes : {16, 64, 256, 1024}) {
        const int threads = lanes > 256 ? lanes : 256, at_a_time = threads / lanes, rows = yan::norm_rows_per_launch(threads, at_a_time);
        std::printf("%d %d %d\\n", threads, at_a_time, rows);
    }
}
""")
    assert len(out) == 4
    for threads, at_a_time, rows in (map(int, line.split()) for line in out):
        assert rows % (8 * at_a_time) == 0 and (1 << 32) - 16 * threads <= rows // at_a_time * threads < 1 << 32 and rows < 1 << 31


def test_layout_asks_for_the_workspace_that_its_launch_wants(tmp_path, monkeypatch):
    """Of any batch that is documented, the tables of which pass 2 GiB at the end of the range."""
    asked = []
    monkeypatch.setattr(moe, 'assert_on_current_device', lambda *_: None)
    monkeypatch.setattr(moe, 'current_raw_stream', lambda: 0)
    monkeypatch.setattr(moe, 'remember_new', lambda *_: None)
    monkeypatch.setattr(moe, '_run', lambda plan, includes, args: asked.append(args) or ('', None, args))
    cases = [(0, 4, 2), (1024, 8, 256), (1025, 8, 256), (1 << 25, 16, 1024), ((1 << 25) + 3, 16, 1024), (moe.MAX_PAIRS // 16, 16, 1024), (moe.MAX_PAIRS, 1, 7)]
    for tokens, top_k, experts in cases:
        yan.moe_ragged_layout(torch.empty(tokens, top_k, dtype=torch.int32, device='meta'), experts)
    out = _host(tmp_path, """
#include "moe/layout.hpp"
#include <cstdio>
int main() {
    long long pairs;
    int experts;
    while (std::scanf("%lld %d", &pairs, &experts) == 2) std::printf("%d\\n", yan::moe_layout_workspace_numbers(pairs, experts));
}
""", '\n'.join(f'{tokens * top_k} {experts}' for tokens, top_k, experts in cases))
    assert max(map(int, out)) > 1 << 30
    for args, numbers in zip(asked, map(int, out)):
        workspace, said = args[4], args[5]
        assert said == numbers and (numbers == 0 or (workspace.numel() == numbers and workspace.dtype == torch.int32))


def test_the_walk_of_large_tiles_has_every_output_once(tmp_path):
    """Slots to tiles of runs of rows and columns, halves of a last round among them: every row of every group meets every column once, whatever the groups, the columns and the
    workgroups (which group a run is of, a wave's look-up on the device, is a loop here)."""
    cases, rng = [], random.Random(5)
    for _ in range(400):
        groups = rng.choice([1, 2, 5, 16, 70])
        counts = [rng.choice([0, 1, 127, 128, 129, 256, 257, rng.randint(0, 700), rng.randint(0, 3000) if groups < 16 else 300]) for _ in range(groups)]
        cases.append((rng.choice([8, 256, 264, 1000, 2048, 4096]), rng.choice([1, 3, 8, 16, 24, 64, 128, 256]), counts))
    out = _host(tmp_path, """
#include "gemm/grouped16.hpp"
#include <cstdio>
#include <vector>
int main() {
    int n, workgroups, groups;
    while (std::scanf("%d %d %d", &n, &workgroups, &groups) == 3) {
        std::vector<int> lo(groups + 1), before(groups + 1);
        for (int g = 0; g < groups; ++g) {
            int rows;
            if (std::scanf("%d", &rows) != 1) return 1;
            lo[g + 1] = lo[g] + rows, before[g + 1] = before[g] + yan::ceil_div(rows, 256);
        }
        const yan::XcdTileScheduler<> sched(before[groups], n, 1, 256);
        const yan::HalvedRound walk(sched.grid_size(), workgroups, true);
        std::vector<int> seen(size_t(lo[groups]) * sched.tiles_n);
        int halves = 0, bad = 0;
        for (int slot = 0; slot < walk.all; ++slot) {
            const int behind = slot - walk.whole, position = sched.dealt_position(behind < 0 ? slot : walk.tile_behind(behind));
            if (position < 0) continue;
            int g = 0;
            while (before[g + 1] <= position / sched.tiles_n) ++g;
            const yan::RunOfGroup at(position - before[g] * sched.tiles_n, before[g + 1] - before[g], sched.tiles_n);
            const int from = lo[g] + at.run * 256 + (walk.is_lower(behind) ? 128 : 0), upto = std::min(from + (behind < 0 ? 256 : 128), lo[g + 1]);
            halves += behind >= 0;
            bad += at.column < 0 || at.column >= sched.tiles_n || at.run < 0 || at.run >= before[g + 1] - before[g];
            for (int r = from; r < upto && !bad; ++r) ++seen[size_t(r) * sched.tiles_n + at.column];
        }
        for (const int times : seen) bad += times != 1;
        std::printf("%d %d\\n", bad, halves);
    }
}
""", '\n'.join(f'{n} {workgroups} {len(counts)} ' + ' '.join(map(str, counts)) for n, workgroups, counts in cases))
    bad, halves = zip(*(map(int, line.split()) for line in out))
    assert len(out) == len(cases) and not any(bad)
    assert any(halves) and not all(halves)


def test_norm_gradients_of_the_widest_rows_use_hardly_any_scratch(tmp_path):
    """Of every combination of types with both gradients asked for: none, but 20 bytes of a lane where h and the weight are fp32."""
    types = (torch.bfloat16, torch.float32)

    def scratch(case):
        _, keys, arg_defs, template = norm.norm_backward_kernel_plan(*case, *norm.norm_backward_lanes(norm.MAX_COLUMNS), True, True)
        stem = '_'.join(str(t).split('.')[1] for t in case)
        src, asm = tmp_path / f'{stem}.cu', tmp_path / f'{stem}.s'
        src.write_text(generate(norm.includes, arg_defs, cpp_format(template, dict(keys))))
        flags = [f for f in get_compile_flags() if f not in ('-shared', '-fPIC')]
        subprocess.check_call([get_hipcc_compiler()[0], '-x', 'hip', '--cuda-device-only', '-S', *flags, f'-I{get_jit_include_dir()}', str(src), '-o', str(asm)])
        return max(int(n) for n in re.findall(r'private_segment_fixed_size: *(\d+)', asm.read_text()))

    cases = list(itertools.product(types, types, types))
    with ThreadPoolExecutor(max_workers=4) as pool:
        for (g, h, w), size in zip(cases, pool.map(scratch, cases)):
            assert size <= (20 if h == w == torch.float32 else 0), (g, h, w)
