// Products of 16-bit operands (bf16 or fp16), group by group, on groups of any number of rows: the experts' products of a layer that is not quantised,
// forward, for the gradient of the rows and for the gradient of the weights. offsets [groups + 1], on the device: group g has rows offsets[g] .. offsets[g + 1] - 1.
//
//   NT   out[r, j]    = sum_t lhs[s(r), t] rhs[g, j, t]      rows r of group g, s(r) = source[r] or r itself
//   NN   out[r, j]    = sum_t lhs[r, t]    rhs[g, t, j]
//   TN   out[g, i, j] (+)= sum_r lhs[r, i] rhs[s(r), j]      over the rows r of group g, fp32
// fp32 sums from the first k-tile to the last; a row whose source is none is a row of zeros.
//
// Two kinds of operand. A plain one has the contraction along its rows: its k-tiles are staged and read as in the other GEMMs (tile_io.hpp). A turned one has the
// contraction across its rows (the weights of NN, both sides of TN): its k-tile is 64 rows of as many columns as the tile has, and a fragment, eight consecutive k of one
// column, comes out of LDS by ds_read_b64_tr_b16, which hands lane i of 16 column i of four rows by sixteen columns. No operand is transposed in memory.
//
// What does not exist is never read: rows behind a group's last one (NT, NN), columns behind a matrix' last one (a turned operand) and k behind the contraction's end
// have the last one that exists copied in their place, so that every copy is within its operand and no copy is out of range for all its lanes. The former
// are not stored. The latter are made zeros in LDS by the wave that copied them, in front of the barrier behind which they are read.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "utils.hpp"
#include "mfma_utils.hpp"
#include "scheduler.hpp"
#include "tile_io.hpp"

namespace yan {

enum class Grouped { NT, NN, TN };

struct GroupedProblem {
    const uint8_t *lhs, *rhs;
    void* out;
    const int *offsets, *source;
    int m, n, k;                // NT, NN: out [m, n], contraction over k; TN: out [groups, m, n], contraction over the rows of both, of which offsets speak
    int rows;                   // rows that offsets speak of: m, or of TN lhs' rows
    int source_rows;            // rows of the operand that is gathered
    int groups;
    bool accumulate;            // TN
};

template <typename Elem> struct Mfma16;
template <> struct Mfma16<__bf16> : MfmaBF16_16x16x32 {};
template <> struct Mfma16<_Float16> : MfmaF16_16x16x32 {};

constexpr int kDepth = 64;              // of a k-tile: 128 bytes of a plain operand's rows

// Rows of group g. Offsets are the caller's, on the device: whatever they hold, the range lies inside of the rows.
__device__ __forceinline__ void grouped_range(const GroupedProblem& p, int g, int& lo, int& hi) {
    lo = min(max(p.offsets[g], 0), p.rows);
    hi = min(max(p.offsets[g + 1], lo), p.rows);
}

// A run of up to BLOCK_M rows of one group, and how many such runs the groups have: a wave looks at 64 groups at a time.
struct RowTile {
    int group, row0, rows;
};
template <int BLOCK_M>
__device__ __forceinline__ int count_row_tiles(const GroupedProblem& p, int lane, int* groups_with_rows) {
    int tiles = 0, with_rows = 0;
    for (int g = lane; g < p.groups; g += kWaveSize) {
        int lo, hi;
        grouped_range(p, g, lo, hi);
        tiles += ceil_div(hi - lo, BLOCK_M);
        with_rows += hi > lo;
    }
#pragma unroll
    for (int d = 1; d < kWaveSize; d *= 2) {
        tiles += __shfl_xor(tiles, d, kWaveSize);
        with_rows += __shfl_xor(with_rows, d, kWaveSize);
    }
    *groups_with_rows = __builtin_amdgcn_readfirstlane(with_rows);
    return __builtin_amdgcn_readfirstlane(tiles);
}
template <int BLOCK_M>
__device__ __forceinline__ RowTile find_row_tile(const GroupedProblem& p, int tile, int lane) {
    int before = 0;
    for (int g0 = 0; g0 < p.groups; g0 += kWaveSize) {
        int lo = 0, hi = 0;
        if (g0 + lane < p.groups) grouped_range(p, g0 + lane, lo, hi);
        const int tiles = ceil_div(hi - lo, BLOCK_M);
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < kWaveSize; d *= 2) {
            const int below = __shfl_up(sum, d, kWaveSize);
            if (lane >= d) sum += below;
        }
        const unsigned long long behind = __ballot(before + sum > tile);
        if (behind) {
            const int at = __builtin_ctzll(behind);
            const int first = before + __builtin_amdgcn_readlane(sum - tiles, at), start = __builtin_amdgcn_readlane(lo, at), end = __builtin_amdgcn_readlane(hi, at);
            const int row0 = start + (tile - first) * BLOCK_M;
            return {g0 + at, row0, min(BLOCK_M, end - row0)};
        }
        before += __builtin_amdgcn_readlane(sum, kWaveSize - 1);
    }
    return {0, 0, 0};
}

// Bytes from `from` on that a descriptor of at most 2 GiB may reach.
__device__ __forceinline__ uint32_t reach(long long bytes) { return bytes < (long long)kOutOfRange ? uint32_t(bytes) : kOutOfRange; }

// Copies of a plain operand's k-tiles, DIM rows of 128 bytes: instruction j of wave w has rows 8 (4 j + w) .. + 7.
template <int DIM>
struct PlainCopies {
    static constexpr int PASSES = DIM / 32;
    uint32_t voff[4];       // (a plain number: with PASSES the compiler leaves out the host side of a kernel that is launched)
    static_assert(PASSES <= 4);
    int chunk;              // of its row that this lane has

    // `row_of(r)`: which row of the descriptor stands for row r of the tile
    template <typename RowOf>
    __device__ __forceinline__ void aim(uint32_t ld_bytes, int wave, int lane, RowOf&& row_of) {
        const int sub = lane >> 3;
        chunk = (lane & 7) ^ sub ^ (wave & 1);
#pragma unroll
        for (int j = 0; j < PASSES; ++j) voff[j] = uint32_t(row_of((j * 4 + wave) * 8 + sub)) * ld_bytes + chunk * kChunk;
    }
    // k-tile `kt`, of which `chunks` chunks a row exist
    __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t rsrc, uint8_t* tile, int kt, int chunks, int wave) const {
        const uint32_t back = chunk < chunks ? 0u : uint32_t(chunk) * kChunk;
#pragma unroll
        for (int j = 0; j < PASSES; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, YAN_LDS_PTR(tile + (j * 4 + wave) * 8 * kRowBytes), kChunk, voff[j] - back, kt * kRowBytes, 0, 0);
    }
    __device__ __forceinline__ void clear(uint8_t* tile, int chunks, int wave, int lane) const {
        if (chunk < chunks) return;
#pragma unroll
        for (int j = 0; j < PASSES; ++j) *reinterpret_cast<i32x4*>(tile + (j * 4 + wave) * 8 * kRowBytes + lane * kChunk) = i32x4{0, 0, 0, 0};
    }
};

// A turned operand's k-tile in LDS: 64 rows of DIM columns, pairs of 16-byte chunks in place pair ^ spread(row), so that the four rows by 32 bytes that 16 lanes read at
// a time, and those of their neighbours, lie in different banks.
template <int DIM>
struct Turned {
    static constexpr int ROW_BYTES = DIM * 2, CHUNKS = DIM / 8;
    __device__ __forceinline__ static int spread(int row) { return ((row & 3) | ((row >> 2) & 12)) & (CHUNKS / 2 - 1); }
    // where lane `lane` reads of rows 16 g + i / 4 of the tile, for column atom 0; atom a: xor 32 a; rows 4 and 8 further on: + 4, 8 ROW_BYTES
    __device__ __forceinline__ static int lane_offset(int lane) {
        const int g = lane / 16, i = lane % 16, row = 16 * g + i / 4;
        return row * ROW_BYTES + spread(row) * 32 + i % 4 * 8;
    }
};

// Copies of a turned operand's k-tiles: instruction j of wave w has ROWS rows from ROWS (4 j + w) on. The descriptor starts at the k-tile's first row, or at the operand's if rows
// are gathered, and at the tile's first column, of which `columns` exist (a multiple of 8).
template <int DIM>
struct TurnedCopies {
    static constexpr int PASSES = DIM / 32, CHUNKS = Turned<DIM>::CHUNKS, ROWS = 1024 / Turned<DIM>::ROW_BYTES;
    static_assert(PASSES <= 4);
    uint32_t column[4];                 // byte offset of this lane's columns in their row
    int row_in;

    __device__ __forceinline__ int row(int j, int wave) const { return (j * 4 + wave) * ROWS + row_in; }
    __device__ __forceinline__ void aim(int columns, int wave, int lane) {
        row_in = lane / CHUNKS;
#pragma unroll
        for (int j = 0; j < PASSES; ++j) column[j] = uint32_t(min((lane % CHUNKS) ^ (Turned<DIM>::spread(row(j, wave)) << 1), columns / 8 - 1)) * kChunk;
    }
    // `row_of(r)`: which row of the descriptor stands for row r of the k-tile
    template <typename RowOf>
    __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t rsrc, uint8_t* tile, uint32_t ld_bytes, int wave, RowOf&& row_of) const {
#pragma unroll
        for (int j = 0; j < PASSES; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, YAN_LDS_PTR(tile + (j * 4 + wave) * 1024), kChunk, uint32_t(row_of(j, row(j, wave))) * ld_bytes + column[j], 0, 0, 0);
    }
    template <typename Bad>
    __device__ __forceinline__ void clear(uint8_t* tile, int wave, int lane, Bad&& bad) const {
#pragma unroll
        for (int j = 0; j < PASSES; ++j)
            if (bad(j, row(j, wave))) *reinterpret_cast<i32x4*>(tile + (j * 4 + wave) * 1024 + lane * kChunk) = i32x4{0, 0, 0, 0};
    }
};

// Eight consecutive k of one column out of a turned k-tile.
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <typename Frag, int DIM>
__device__ __forceinline__ Frag read_turned(const uint8_t* at) {
    typedef __attribute__((address_space(3))) s16x4* LdsPtr;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsPtr>(YAN_LDS_PTR(at)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsPtr>(YAN_LDS_PTR(at + 4 * Turned<DIM>::ROW_BYTES)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(Frag, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
}

// Tiles of 128 x 128 and less: 4 waves, a ring of STAGES k-tiles, one tile a workgroup, or a walk under a cap. Two workgroups or more a compute unit hide each other's waits.
template <typename Elem, Grouped MODE, int BLOCK_M, int BLOCK_N, int STAGES, bool GATHER>
__global__ void __launch_bounds__(256, 2)
grouped16_kernel(GroupedProblem p, int slots) {
    constexpr bool TURN_A = MODE == Grouped::TN, TURN_B = MODE != Grouped::NT;
    constexpr int WAVES_M = BLOCK_M >= 64 ? 2 : 1, WAVES_N = 4 / WAVES_M, WTM = BLOCK_M / WAVES_M, WTN = BLOCK_N / WAVES_N, TM = WTM / 16, TN = WTN / 16;
    static_assert(BLOCK_M % 32 == 0 && BLOCK_N % 32 == 0 && WTM % 16 == 0 && WTN % 16 == 0 && !(GATHER && MODE == Grouped::NN));
    using CopiesA = std::conditional_t<TURN_A, TurnedCopies<BLOCK_M>, PlainCopies<BLOCK_M>>;
    using CopiesB = std::conditional_t<TURN_B, TurnedCopies<BLOCK_N>, PlainCopies<BLOCK_N>>;
    using Frag = typename Mfma16<Elem>::Frag;
    // TN: the sources of a later k-tile come with a k-tile, each wave its own
    constexpr bool SOURCES = GATHER && MODE == Grouped::TN;
    constexpr int A_BYTES = BLOCK_M * kRowBytes, STAGE_BYTES = (BLOCK_M + BLOCK_N) * kRowBytes, NUM_COPIES = CopiesA::PASSES + CopiesB::PASSES + (SOURCES ? 1 : 0);
    static_assert((STAGES - 1) * NUM_COPIES <= 63);
    __shared__ __attribute__((aligned(1024))) uint8_t ring[STAGES * STAGE_BYTES];
    __shared__ __attribute__((aligned(256))) int ring_sources[SOURCES ? STAGES * 4 * kDepth : 1];

    const int lane = get_lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int wn = wave % WAVES_N, wm = wave / WAVES_N, g = lane / 16, col = lane % 16;
    int with_rows = 0;
    const int row_tiles = MODE == Grouped::TN ? 0 : count_row_tiles<BLOCK_M>(p, lane, &with_rows);
    XcdTileScheduler<> sched(MODE == Grouped::TN ? p.m : row_tiles * BLOCK_M, p.n, BLOCK_M, BLOCK_N);
    if (MODE != Grouped::TN) sched.fit_bands_to_groups(with_rows ? row_tiles / with_rows : 1);
    const int per_group = sched.grid_size();
    if (MODE != Grouped::TN) slots = per_group;
    for (int slot = blockIdx.x; slot < slots; slot += gridDim.x) {
        const int tile_group = MODE == Grouped::TN ? slot / per_group : 0;
        const TileCoord tile = sched.tile_of(slot - tile_group * per_group);
        if (!tile.valid) continue;
        const int n0 = tile.n_idx * BLOCK_N, cols = min(BLOCK_N, p.n - n0);
        // rows m0 .. m0 + rows_m - 1 of the output; contraction from k0 on over `depth`
        int group, m0, rows_m, k0, depth;
        if constexpr (MODE == Grouped::TN) {
            group = tile_group, m0 = tile.m_idx * BLOCK_M, rows_m = min(BLOCK_M, p.m - m0);
            int hi;
            grouped_range(p, group, k0, hi);
            depth = hi - k0;
            if (p.accumulate && depth == 0) continue;
        } else {
            const RowTile t = find_row_tile<BLOCK_M>(p, tile.m_idx, lane);
            group = t.group, m0 = t.row0, rows_m = t.rows, k0 = 0, depth = p.k;
        }
        // the ring is used again: everybody is out of it
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");

        const int count = ceil_div(depth, kDepth), last_depth = depth - (count - 1) * kDepth;
        const auto depth_of = [&](int kt) { return kt + 1 < count ? kDepth : last_depth; };
        // operands with the contraction along their rows: descriptors from the tile's first row on
        const uint32_t ld_a = uint32_t(MODE == Grouped::TN ? p.m : p.k) * 2, ld_b = uint32_t(MODE == Grouped::NT ? p.k : p.n) * 2;
        const uint8_t* const base_b = MODE == Grouped::TN ? p.rhs : p.rhs + size_t(group) * p.n * p.k * 2;
        __amdgpu_buffer_rsrc_t rsrc_a, rsrc_b;
        CopiesA copies_a;
        CopiesB copies_b;
        if constexpr (TURN_A) {
            copies_a.aim(rows_m, wave, lane);
        } else if constexpr (GATHER) {
            rsrc_a = make_rsrc(p.lhs, reach((long long)p.source_rows * ld_a));
            copies_a.aim(ld_a, wave, lane, [&](int r) {
                const int s = p.source[m0 + min(r, rows_m - 1)];
                return uint32_t(s) < uint32_t(p.source_rows) ? s : 0;
            });
        } else {
            rsrc_a = make_rsrc(p.lhs + size_t(m0) * ld_a, uint32_t(rows_m) * ld_a);
            copies_a.aim(ld_a, wave, lane, [&](int r) { return min(r, rows_m - 1); });
        }
        if constexpr (TURN_B) {
            copies_b.aim(cols, wave, lane);
            if constexpr (SOURCES) rsrc_b = make_rsrc(p.rhs + n0 * 2, reach((long long)p.source_rows * ld_b - n0 * 2));
        } else {
            rsrc_b = make_rsrc(base_b + size_t(n0) * ld_b, uint32_t(cols) * ld_b);
            copies_b.aim(ld_b, wave, lane, [&](int r) { return min(r, cols - 1); });
        }
        // of the gathered rows of the k-tiles under way, a bit a pass and 8 a k-tile, the youngest lowest: they are none
        [[maybe_unused]] uint32_t none = 0;
        const __amdgpu_buffer_rsrc_t rsrc_s = make_rsrc(SOURCES ? p.source + k0 : nullptr, uint32_t(SOURCES ? depth : 0) * 4);
        auto copy = [&](int kt, int st, auto from_memory) __attribute__((always_inline)) {
            if (kt >= count) return;
            uint8_t* const stage = ring + st * STAGE_BYTES;
            const int here = depth_of(kt);
            [[maybe_unused]] int sources[CopiesB::PASSES];
            if constexpr (SOURCES) {
                none <<= 8;
#pragma unroll
                for (int j = 0; j < CopiesB::PASSES; ++j) {
                    int r = 0;
                    if constexpr (TURN_B) r = min(copies_b.row(j, wave), here - 1);
                    const int s = decltype(from_memory)::value ? p.source[k0 + kt * kDepth + r] : ring_sources[(st * 4 + wave) * kDepth + r];
                    const bool there = uint32_t(s) < uint32_t(p.source_rows);
                    sources[j] = there ? s : 0;
                    none |= there ? 0u : 1u << j;
                }
            }
            if constexpr (TURN_A) {
                const long long left = (long long)(p.rows - k0 - kt * kDepth) * ld_a - m0 * 2;
                copies_a.issue(make_rsrc(p.lhs + size_t(k0 + kt * kDepth) * ld_a + m0 * 2, reach(left)), stage, ld_a, wave, [&](int, int r) { return min(r, here - 1); });
            } else {
                copies_a.issue(rsrc_a, stage, kt, here / 8, wave);
            }
            if constexpr (SOURCES) {
                copies_b.issue(rsrc_b, stage + A_BYTES, ld_b, wave, [&](int j, int) { return sources[j]; });
                // those of the k-tile that takes this stage next
                const int next = min((kt + STAGES) * kDepth + lane, depth - 1);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_s, YAN_LDS_PTR(ring_sources + (st * 4 + wave) * kDepth), 4, next * 4, 0, 0, 0);
            } else if constexpr (TURN_B) {
                const long long left = (long long)((MODE == Grouped::TN ? p.rows : p.k) - k0 - kt * kDepth) * ld_b - n0 * 2;
                copies_b.issue(make_rsrc(base_b + size_t(k0 + kt * kDepth) * ld_b + n0 * 2, reach(left)), stage + A_BYTES, ld_b, wave, [&](int, int r) { return min(r, here - 1); });
            } else {
                copies_b.issue(rsrc_b, stage + A_BYTES, kt, here / 8, wave);
            }
        };
        // makes zeros of what a k-tile has copied of what does not exist, by the wave that did; `age`: copied so many k-tiles ago
        auto clear = [&](int kt, int st, int age) __attribute__((always_inline)) {
            uint8_t* const stage = ring + st * STAGE_BYTES;
            const int here = depth_of(kt);
            bool any = here < kDepth;
            if constexpr (SOURCES) any |= __ballot(((none >> (8 * age)) & 255) != 0) != 0;
            if (!any) return;
            if constexpr (TURN_A) copies_a.clear(stage, wave, lane, [&](int, int r) { return r >= here; });
            else copies_a.clear(stage, here / 8, wave, lane);
            if constexpr (TURN_B)
                copies_b.clear(stage + A_BYTES, wave, lane, [&](int j, int r) {
                    bool bad = r >= here;
                    if constexpr (SOURCES) bad |= (none >> (8 * age + j)) & 1;
                    return bad;
                });
            else copies_b.clear(stage + A_BYTES, here / 8, wave, lane);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoWaitVm, 0));
        };

        f32x4 acc[TN][TM];
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int plain[2] = {frag_offset<16>(lane, 2 * g), frag_offset<16>(lane, 2 * g + 1)};
        const int turned_a = Turned<BLOCK_M>::lane_offset(lane), turned_b = Turned<BLOCK_N>::lane_offset(lane);
        auto multiply = [&](int st) __attribute__((always_inline)) {
            const uint8_t *const pa = ring + st * STAGE_BYTES, *const pb = pa + A_BYTES;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag fa[TM], fb[TN];
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    if constexpr (TURN_A) fa[j] = read_turned<Frag, BLOCK_M>(pa + 8 * h * Turned<BLOCK_M>::ROW_BYTES + (turned_a ^ ((wm * TM + j) * 32)));
                    else fa[j] = *reinterpret_cast<const Frag*>(pa + (wm * WTM + j * 16) * kRowBytes + plain[h]);
                }
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    if constexpr (TURN_B) fb[i] = read_turned<Frag, BLOCK_N>(pb + 8 * h * Turned<BLOCK_N>::ROW_BYTES + (turned_b ^ ((wn * TN + i) * 32)));
                    else fb[i] = *reinterpret_cast<const Frag*>(pb + (wn * WTN + i * 16) * kRowBytes + plain[h]);
                }
#pragma unroll
                for (int i = 0; i < TN; ++i)
#pragma unroll
                    for (int j = 0; j < TM; ++j) acc[i][j] = Mfma16<Elem>::mma(fb[i], fa[j], acc[i][j]);
            }
        };
        for (int t = 0; t < STAGES - 1; ++t) copy(t, t, std::true_type{});
        int st = 0;
        for (int kt = 0; kt < count; ++kt) {
            if (kt + STAGES - 2 < count) __builtin_amdgcn_s_waitcnt(waitcnt_imm((STAGES - 2) * NUM_COPIES, kNoWaitLgkm));
            else __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, kNoWaitLgkm));
            asm volatile("" ::: "memory");
            // (k-tiles copied behind this one: STAGES - 2, or as many as there are)
            clear(kt, st, min(STAGES - 2, count - 1 - kt));
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const int into = st == 0 ? STAGES - 1 : st - 1;
            // the first k-tile into the last stage finds no sources there
            if (kt == 0) copy(kt + STAGES - 1, into, std::true_type{});
            else copy(kt + STAGES - 1, into, std::false_type{});
            multiply(st);
            __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoWaitVm, 0));         // what this wave reads of the stage is in registers: the next barrier frees it
            st = st + 1 == STAGES ? 0 : st + 1;
        }

        // The 4 registers of atom (i, j) are columns 16 i + 4 g + {0..3} of row 16 j + col of the slab. A wave turns its slab round through LDS and stores 16 bytes a lane.
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if constexpr (MODE == Grouped::TN) {
            // as the FP8 weight gradients: chunk c of a row in slot c ^ row, whole lines
            constexpr int LANES_PER_ROW = WTN / 4, ROWS_PER_STORE = kWaveSize / LANES_PER_ROW, STORES = WTM / ROWS_PER_STORE;
            static_assert(4 * WTM * WTN * 4 <= STAGES * STAGE_BYTES && kWaveSize % LANES_PER_ROW == 0);
            uint8_t* const region = ring + wave * (WTM * WTN * 4);
            const auto place = [](int row, int chunk) { return row * (WTN * 4) + ((chunk ^ (row & (LANES_PER_ROW - 1))) * 16); };
            const int row_in = lane / LANES_PER_ROW, chunk = lane % LANES_PER_ROW, c0 = wn * WTN + 4 * chunk;
            const bool stream_out = size_t(p.groups) * p.m * p.n * 4 > (size_t(32) << 20);
            const uint32_t row_bytes = uint32_t(p.n) * 4;
            const __amdgpu_buffer_rsrc_t rsrc_out = make_rsrc(static_cast<float*>(p.out) + (size_t(group) * p.m + m0) * p.n + n0, uint32_t(rows_m) * row_bytes - uint32_t(n0) * 4);
            const uint32_t to = c0 < cols ? uint32_t(wm * WTM + row_in) * row_bytes + uint32_t(c0) * 4 : kOutOfRange;
            i32x4 held[STORES];
            if (p.accumulate) {
#pragma unroll
                for (int u = 0; u < STORES; ++u) held[u] = __builtin_amdgcn_raw_buffer_load_b128(rsrc_out, to, u * ROWS_PER_STORE * row_bytes, 0);
            }
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int i = 0; i < TN; ++i) *reinterpret_cast<f32x4*>(region + place(16 * j + col, 4 * i + g)) = acc[i][j];
#pragma unroll
            for (int u = 0; u < STORES; ++u) {
                f32x4 v = *reinterpret_cast<const f32x4*>(region + place(u * ROWS_PER_STORE + row_in, chunk));
                if (p.accumulate) v += __builtin_bit_cast(f32x4, held[u]);
                buffer_store_16(__builtin_bit_cast(i32x4, v), rsrc_out, to + u * ROWS_PER_STORE * row_bytes, stream_out);
            }
        } else {
            constexpr int PITCH = WTN * 2 + 16, LANES_PER_ROW = WTN / 8, ROWS_PER_STORE = kWaveSize / LANES_PER_ROW, STORES = ceil_div(WTM, ROWS_PER_STORE);
            static_assert(4 * WTM * PITCH <= STAGES * STAGE_BYTES && kWaveSize % LANES_PER_ROW == 0);
            uint8_t* const region = ring + wave * (WTM * PITCH);
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int i = 0; i < TN; ++i)
                    *reinterpret_cast<decltype(pack4(acc[0][0], Elem{}))*>(region + (16 * j + col) * PITCH + (16 * i + 4 * g) * 2) = pack4(acc[i][j], Elem{});
            const int row_in = lane / LANES_PER_ROW, c = lane % LANES_PER_ROW, c0 = wn * WTN + 8 * c;
            const bool stream_out = size_t(p.m) * p.n * 2 > (size_t(32) << 20);
            const uint32_t row_bytes = uint32_t(p.n) * 2;
            const __amdgpu_buffer_rsrc_t rsrc_out = make_rsrc(static_cast<uint8_t*>(p.out) + (size_t(m0) * p.n + n0) * 2, uint32_t(rows_m) * row_bytes - uint32_t(n0) * 2);
#pragma unroll
            for (int u = 0; u < STORES; ++u) {
                const int row = u * ROWS_PER_STORE + row_in, r = wm * WTM + row;
                const bool mine = row < WTM && r < rows_m && c0 < cols;
                i32x4 v = i32x4{0, 0, 0, 0};
                if (row < WTM) v = *reinterpret_cast<const i32x4*>(region + row * PITCH + c * 16);
                if constexpr (GATHER) {
                    if (mine && uint32_t(p.source[m0 + r]) >= uint32_t(p.source_rows)) v = i32x4{0, 0, 0, 0};
                }
                buffer_store_16(v, rsrc_out, mine ? uint32_t(r) * row_bytes + uint32_t(c0) * 2 : kOutOfRange, stream_out);
            }
        }
    }
}

enum Grouped16Kernel { kGroupedAny, kGrouped128, kGrouped64, kGrouped32 };

// Rows that offsets speak of, and columns of a matrix: less than so many, so that tiles and ranges stay within 32-bit offsets.
constexpr int kGroupedMostRows = 1 << 29, kGroupedMostColumns = 1 << 21;

// lhs, rhs, out as Grouped has them, contiguous, 16-byte aligned; n and k (TN: m and n) multiples of 8. source: [rows] or null; source_rows: rows of the operand that is gathered.
template <typename Elem, Grouped MODE, bool GATHER, Grouped16Kernel KERNEL = kGroupedAny>
inline hipError_t launch_grouped16(const void* lhs, const void* rhs, void* out, const int* offsets, const int* source, int groups, int rows, int m, int n, int k, int source_rows,
                                   bool accumulate, int num_sms, hipStream_t stream) {
    if (groups < 0 || rows < 0 || rows >= kGroupedMostRows || m < 0 || n < 0 || k < 0 || n % 8 != 0 || n >= kGroupedMostColumns) return hipErrorInvalidValue;
    if (MODE == Grouped::TN ? m % 8 != 0 || m >= kGroupedMostColumns : k % 8 != 0 || k >= kGroupedMostColumns || m != rows) return hipErrorInvalidValue;
    if (GATHER && (!source || source_rows < 1 || (long long)source_rows * (MODE == Grouped::TN ? n : k) * 2 >= (long long)kOutOfRange)) return hipErrorInvalidValue;
    if (m == 0 || n == 0 || groups == 0) return hipSuccess;
    if (!out || !offsets || (rows && (MODE == Grouped::TN || k) && (!lhs || !rhs))) return hipErrorInvalidValue;
    const GroupedProblem p{static_cast<const uint8_t*>(lhs), static_cast<const uint8_t*>(rhs), out, offsets, source, m, n, k, rows, source_rows, groups, accumulate};
    const bool capped = num_sms > 0 && num_sms < device_cu_count();
    const auto slots_of = [&](int block_m, int block_n) -> long long {
        if (MODE == Grouped::TN) return (long long)XcdTileScheduler<>(m, n, block_m, block_n).grid_size() * groups;
        // as many runs as the groups' rows can have
        const long long runs = std::min<long long>(m, ((long long)m + (long long)(block_m - 1) * groups) / block_m);
        return ceil_div<long long>(runs * ceil_div(n, block_n), kNumXCD) * kNumXCD;
    };
    const auto launch = [&](auto kernel, int block_m, int block_n) {
        const long long slots = slots_of(block_m, block_n);
        if (slots >= 1ll << 24) return hipErrorInvalidValue;          // a launch has less than 2^32 threads
        hipLaunchKernelGGL(kernel, dim3(uint32_t(capped ? capped_grid(int(slots), num_sms, device_cu_count()) : slots)), dim3(256), 0, stream, p, int(slots));
        return hipGetLastError();
    };
    Grouped16Kernel which = KERNEL;
    if (which == kGroupedAny) {
        const long long each = MODE == Grouped::TN ? m : rows / groups;
        which = MODE != Grouped::TN && each <= 24 ? kGrouped32 : slots_of(128, 128) >= device_cu_count() ? kGrouped128 : kGrouped64;
    }
    switch (which) {
        case kGrouped32: return launch(grouped16_kernel<Elem, MODE, 32, 128, 4, GATHER>, 32, 128);
        case kGrouped64: return launch(grouped16_kernel<Elem, MODE, 64, 64, 4, GATHER>, 64, 64);
        default: return launch(grouped16_kernel<Elem, MODE, 128, 128, 2, GATHER>, 128, 128);
    }
}

} // namespace yan
