// Products of 16-bit operands (bf16 or fp16), group by group, on groups of any number of rows: the experts' products of a layer that is not quantised,
// forward, for the gradient of the rows and for the gradient of the weights. offsets [groups + 1], on the device: group g has rows offsets[g] .. offsets[g + 1] - 1.
//
//   NT   out[r, j]    = sum_t lhs[s(r), t] rhs[g, j, t]      rows r of group g, s(r) = source[r] or r itself
//   NN   out[r, j]    = sum_t lhs[r, t]    rhs[g, t, j]
//   TN   out[g, i, j] (+)= sum_r lhs[r, i] rhs[s(r), j]      over the rows r of group g, fp32
// fp32 sums from the first k-tile to the last. A row whose source is none is a row of zeros of NT's out, and no row of TN's sum, whatever the other operand holds.
//
// Two kinds of operand. A plain one has the contraction along its rows: its k-tiles are staged and read as in the other GEMMs (tile_io.hpp). A turned one has the
// contraction across its rows (the weights of NN, both sides of TN): its k-tile is 64 rows of as many columns as the tile has, and a fragment, eight consecutive k of one
// column, comes out of LDS by ds_read_b64_tr_b16, which hands lane i of 16 column i of four rows by sixteen columns. No operand is transposed in memory.
//
// What does not exist is never read: rows behind a group's last one (NT, NN) and columns behind a matrix' last one have the last one that exists copied in their place, and are not
// stored. So has k behind the contraction's end in the ring tiles; the large ones copy what comes next, the next row's k, another group's rows or, of a plain operand's last row, nothing for
// the lanes that are out of the descriptor's range, and a turned operand's last row where that ends. Either way no copy reads outside of its operand, none is out of range for all
// its lanes, and k behind the end is made zeros in LDS by the wave that copied it, in front of the barrier behind which it is read.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>
#include <utility>

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

// Runs of `block_m` rows that ascending offsets cut `rows` rows into at most.
__host__ __device__ inline int most_row_tiles(int rows, int groups, int block_m) {
    const long long runs = ((long long)rows + (long long)(block_m - 1) * groups) / block_m;
    return runs < rows ? int(runs) : rows;
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
    // (offsets that do not ascend could say more, of which there is no end)
    return min(__builtin_amdgcn_readfirstlane(tiles), most_row_tiles(p.rows, p.groups, BLOCK_M));
}
// The group that run `tile` is of: its rows, and the runs of the groups before it.
struct GroupRuns {
    int group, lo, hi, before;
};
template <int BLOCK_M>
__device__ __forceinline__ GroupRuns find_group(const GroupedProblem& p, int tile, int lane) {
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
            return {g0 + at, __builtin_amdgcn_readlane(lo, at), __builtin_amdgcn_readlane(hi, at), before + __builtin_amdgcn_readlane(sum - tiles, at)};
        }
        before += __builtin_amdgcn_readlane(sum, kWaveSize - 1);
    }
    return {0, 0, 0, 0};
}
template <int BLOCK_M>
__device__ __forceinline__ RowTile find_row_tile(const GroupedProblem& p, int tile, int lane) {
    const GroupRuns g = find_group<BLOCK_M>(p, tile, lane);
    const int row0 = g.lo + (tile - g.before) * BLOCK_M;
    return {g.group, row0, min(BLOCK_M, g.hi - row0)};
}

// Bytes, not less than none, that a descriptor of at most 2 GiB may reach. (In halves: the scalar unit does not compare numbers of 64 bits, and a descriptor that is not in
// scalar registers is taken there lane by lane, in front of every copy.)
__host__ __device__ __forceinline__ uint32_t reach(long long bytes) {
    const uint32_t upper = uint32_t((unsigned long long)bytes >> 32), lower = uint32_t(bytes);
    return upper != 0 || lower > kOutOfRange ? kOutOfRange : lower;
}
// The same of a descriptor that starts kCopyBias bytes early, as the large tiles' do: the bias comes on top, so that `bytes` of up to 2 GiB are reached to the last one.
constexpr uint32_t kCopyBias = 3 * 1024;
__host__ __device__ __forceinline__ uint32_t biased_reach(long long bytes) { return reach(bytes) + kCopyBias; }

// Whether whole k-tiles of a turned operand of `k` rows, with `left` such operands up to the last one, go beyond the end of that: of the last one itself where k is no whole number of
// them, and of some before it where k is a few rows. (Eight operands have at least as many rows as the k-tiles of the first, k being a multiple of 8; more would pass 32 bits.)
__host__ __device__ __forceinline__ bool weights_end_inside(int left, int k) { return (left < 8 ? left : 8) * k < ceil_div(k, kDepth) * kDepth; }

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

// Eight consecutive k of one column out of a turned k-tile. (Of a read of LDS of which nothing is known the compiler thinks that it may be of what any copy under way brings, and
// waits for all of them in front of it; a restricted pointer is something known. What has landed when is the kernels' own business.)
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <typename Frag, int DIM>
__device__ __forceinline__ Frag read_turned(const uint8_t* __restrict__ at) {
    typedef __attribute__((address_space(3))) s16x4* LdsPtr;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at + 4 * Turned<DIM>::ROW_BYTES));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(Frag, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
}

// One of the two reads of that.
template <typename Frag>
__device__ __forceinline__ void read_turned_part(Frag& f, const uint8_t* __restrict__ at, int part) {
    typedef __attribute__((address_space(3))) s16x4* LdsPtr;
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at));
    s16x8 all = __builtin_bit_cast(s16x8, f);
    if (part == 0) all[0] = v[0], all[1] = v[1], all[2] = v[2], all[3] = v[3];
    else all[4] = v[0], all[5] = v[1], all[6] = v[2], all[7] = v[3];
    f = __builtin_bit_cast(Frag, all);
}

typedef int i32x16_unaligned __attribute__((ext_vector_type(16), aligned(4)));

// f(0), f(1), ... f(N - 1), each with its number as a constant.
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    [&]<int... I>(std::integer_sequence<int, I...>) __attribute__((always_inline)) { (f(std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, N>{});
}

// Tiles of 128 x 128 and less: 4 waves, a ring of STAGES k-tiles, one tile a workgroup, or a walk under a cap. Two workgroups a compute unit hide each other's waits.
// For few rows a group, where the weights' bytes bound the product (or those of their gradients): 32 experts of 8 rows, 4096 x 7168, bf16 (1.88 GB): 300 us, 6.3 TB/s. Gradients
// added to 32 experts of 2048 x 1024 for 62 rows each (549 MB): 90 us, 6.1 TB/s.
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
    XcdTileScheduler<> sched(MODE == Grouped::TN ? p.m : row_tiles, p.n, MODE == Grouped::TN ? BLOCK_M : 1, BLOCK_N);
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
            // (a row without a source counts for nothing, whatever the other operand has there: both have the same rows in the same lanes)
            static_assert(!SOURCES || BLOCK_M == BLOCK_N);
            const auto bad = [&](int j, int r) { return r >= here || (SOURCES && ((none >> (8 * age + j)) & 1)); };
            if constexpr (TURN_A) copies_a.clear(stage, wave, lane, bad);
            else copies_a.clear(stage, here / 8, wave, lane);
            if constexpr (TURN_B) copies_b.clear(stage + A_BYTES, wave, lane, bad);
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
                for (int u = 0; u < STORES; ++u) held[u] = __builtin_amdgcn_raw_buffer_load_b128(rsrc_out, to + u * ROWS_PER_STORE * row_bytes, 0, 0);
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

// The groups' rows cut into runs of BLOCK_M, as count_row_tiles and find_group have them, with the first 64 groups in registers: a walk that looks a tile up among its
// copies does not wait for memory.
template <int BLOCK_M>
struct RowRuns {
    int lo, hi, upto;               // of group `lane`: its rows, and the runs up to its last
    __device__ __forceinline__ void init(const GroupedProblem& p, int lane) {
        lo = hi = 0;
        if (lane < p.groups) grouped_range(p, lane, lo, hi);
        upto = ceil_div(hi - lo, BLOCK_M);
#pragma unroll
        for (int d = 1; d < kWaveSize; d *= 2) {
            const int below = __shfl_up(upto, d, kWaveSize);
            if (lane >= d) upto += below;
        }
    }
    __device__ __forceinline__ GroupRuns find(const GroupedProblem& p, int tile, int lane) const {
        const unsigned long long behind = __ballot(upto > tile);
        if (!behind) return find_group<BLOCK_M>(p, tile, lane);
        const int at = __builtin_ctzll(behind);
        const int start = __builtin_amdgcn_readlane(lo, at), end = __builtin_amdgcn_readlane(hi, at);
        return {at, start, end, __builtin_amdgcn_readlane(upto, at) - ceil_div(end - start, BLOCK_M)};
    }
};

// Tiles of 256 x 256 on 4 waves, one a SIMD, each with 128 x 128 outputs in 16x16x32 MFMAs, its sums in the accumulation registers: the design of dense_gemm_body_4w
// (bf16_gemm.hpp). LDS is a ring of five units of 32 KB, a unit being one operand's k-tile; the fragments of half a k-tile are read while the half before it is
// multiplied; copies run two k-tiles ahead of the MFMAs, along K and on into the next tile of a persistent walk, whose first k-tiles are under way when this one's sums leave.
// What is different:
//   * row atoms alternate between the two waves that share a tile's rows, so that a tile at a group's end has them split evenly; one with up to 128 rows (FLAT) runs half of
//     the MFMAs and copies half of the rows. Groups end in the middle of a tile, on average; with 512 rows a group whole tiles would be a quarter more work.
//   * lane offsets of the copies are worked out anew for tiles that are not whole (rows that stand in for those that do not exist) and for gathered rows;
//   * descriptors of turned operands move on with the k-tile, so that ranges may be of any length;
//   * any number of k-tiles, one for instance: the copies' place in the walk is its own.
// Bound by the MFMAs for long groups: 16384 rows of one group x 4096 x 4096 1535 TFLOP/s (dense_gemm_body_4w 1554), NN 1430, TN 1519; of 16 equal groups 1390. Ragged ones lose what
// their last tiles hold too little, 6 to 9 % of the MFMAs' rows, and more by a walk that gives every workgroup as many tiles whatever their heights: the busiest has 16 to 29 % more rows of
// MFMAs than the mean in 32768 rows of 64 experts x 2048 x 7168, gathered: 867 to 970 us by how the router spreads them, 990 to 1110 TFLOP/s. TN writes fp32: of 16 experts x
// 4096 x 7168 (1.88 GB) 6144 rows take 540 to 607 us, 250 of MFMAs and the stores behind them.
struct GroupedTile {
    int slot, group, m0, rows, n0, cols, k0, depth;         // depth 0: none
    __device__ __forceinline__ int count() const { return ceil_div(depth, kDepth); }
    // In the lanes of one register, for tiles that wait for their turn.
    __device__ __forceinline__ int packed(int lane) const {
        return lane & 4 ? (lane & 2 ? (lane & 1 ? depth : k0) : (lane & 1 ? cols : n0)) : (lane & 2 ? (lane & 1 ? rows : m0) : (lane & 1 ? group : slot));
    }
    __device__ __forceinline__ static GroupedTile unpacked(int v) {
        const auto lane = [&](int i) { return __builtin_amdgcn_readlane(v, i); };
        return {lane(0), lane(1), lane(2), lane(3), lane(4), lane(5), lane(6), lane(7)};
    }
};

// The slots of the large tiles' walk. A last round of tiles for at most half of the workgroups is dealt out in halves of 128 rows, two slots a tile on one XCD (4 groups of 285 rows,
// 4096 x 7168, 96 tiles 126 -> 78 us; 16 of 364, 7168 x 4096 back, 868 tiles 368 -> 356).
struct HalvedRound {
    int whole, all;                 // slots of whole tiles, and all of them
    __host__ __device__ HalvedRound(int slots, int workgroups, bool may) {
        const int last_round = slots % workgroups;
        const bool halves = may && 2 * last_round <= workgroups && last_round % kNumXCD == 0;
        whole = halves ? slots - last_round : slots, all = halves ? slots + last_round : slots;
    }
    // A slot that is `behind` the whole tiles' (not below 0) has a half of the tile of this slot, the lower one or the upper.
    __host__ __device__ int tile_behind(int behind) const { return whole + behind / (2 * kNumXCD) * kNumXCD + behind % kNumXCD; }
    __host__ __device__ static bool is_lower(int behind) { return behind >= 0 && behind / kNumXCD % 2; }
};

// A group's tiles follow each other, column by column of up to eight runs of rows: its weights are read by one XCD or, column for column, by two. Bands of rows that
// do not end where groups do read most of them twice (16 experts x 7168 x 4096 back, 3967 rows 278 -> 265 us, 6144 rows 380 -> 374; forward, 64 experts x 2048 x 7168, the same).
struct RunOfGroup {
    int run, column;
    __host__ __device__ RunOfGroup(int in_group, int runs, int tiles_n) {
        constexpr int BAND = 8;
        const int band = in_group / (BAND * tiles_n), in_band = in_group - band * BAND * tiles_n, left = runs - band * BAND, height = left < BAND ? left : BAND;
        column = in_band / height;
        run = band * BAND + in_band - column * height;
    }
};

template <typename Elem, Grouped MODE, bool GATHER>
__global__ void __launch_bounds__(256, 1)
grouped16_tall_kernel(GroupedProblem p) {
    constexpr bool TURN_A = MODE == Grouped::TN, TURN_B = MODE != Grouped::NT, SOURCES = GATHER && MODE == Grouped::TN, GATHER_A = GATHER && MODE == Grouped::NT;
    constexpr int BLOCK = 256, TN = 8, TM = 8, UNITS = 5, UNIT_BYTES = BLOCK * kRowBytes, PASSES = 8;
    static_assert(!(GATHER && MODE == Grouped::NN));
    using Frag = typename Mfma16<Elem>::Frag;
    constexpr int ROW_BYTES = Turned<BLOCK>::ROW_BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[UNITS * UNIT_BYTES];

    const int lane = get_lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int wn = wave % 2, wm = wave / 2, g = lane / 16, col = lane % 16;
    RowRuns<BLOCK> runs;
    int with_rows, row_tiles, tiles_m = 1;
    if constexpr (MODE == Grouped::TN) {
        tiles_m = ceil_div(p.m, BLOCK);
        row_tiles = tiles_m * p.groups;
    } else {
        runs.init(p, lane);
        row_tiles = count_row_tiles<BLOCK>(p, lane, &with_rows);
    }
    const int slots = XcdTileScheduler<>(row_tiles, p.n, 1, BLOCK).grid_size();
    const HalvedRound walk(slots, gridDim.x, MODE != Grouped::TN);
    auto tile_at = [&](int slot) __attribute__((always_inline)) {
        // (worked out anew for every tile: a dozen scalar registers less over the k-loop, which has none to spare)
        int rows_anew = row_tiles;
        asm volatile("" : "+s"(rows_anew));
        XcdTileScheduler<> sched(rows_anew, p.n, 1, BLOCK);
        if constexpr (MODE == Grouped::TN) sched.fit_bands_to_groups(tiles_m);
        // Patches of 32 tiles are dealt out to the XCDs: tiles at a group's end take less time than others, groups of TN differ in their depth, and a range of tiles for each XCD would
        // leave some with more work than others (32768 rows of 64 experts x 2048 x 7168 916 -> 886 us, 6144 of 16 x 7168 x 4096 back 401 -> 381).
        const int behind = slot - walk.whole, of_tile = MODE == Grouped::TN || behind < 0 ? slot : walk.tile_behind(behind);
        GroupedTile t{slot, -1, 0, 0, 0, 0, 0, 0};
        if constexpr (MODE == Grouped::TN) {
            const TileCoord c = sched.dealt_band_tile_of(of_tile);
            if (!c.valid) return t;
            t.n0 = c.n_idx * BLOCK;
            t.group = c.m_idx / tiles_m, t.m0 = (c.m_idx - t.group * tiles_m) * BLOCK, t.rows = min(BLOCK, p.m - t.m0);
            int hi;
            grouped_range(p, t.group, t.k0, hi);
            t.depth = hi - t.k0;
        } else {
            const int position = sched.dealt_position(of_tile), tiles_n = sched.tiles_n;
            if (position < 0) return t;
            const GroupRuns g = runs.find(p, position / tiles_n, lane);
            const RunOfGroup at(position - g.before * tiles_n, ceil_div(g.hi - g.lo, BLOCK), tiles_n);
            const int from = g.lo + at.run * BLOCK + (walk.is_lower(behind) ? BLOCK / 2 : 0);
            t.n0 = at.column * BLOCK, t.group = g.group, t.m0 = from, t.rows = min(behind < 0 ? BLOCK : BLOCK / 2, g.hi - from), t.depth = t.rows > 0 ? p.k : 0;
        }
        t.cols = min(BLOCK, p.n - t.n0);
        return t;
    };
    // the next tile of this workgroup's walk, from `slot` on
    auto seek = [&](int slot) __attribute__((always_inline)) {
        for (; slot < walk.all; slot += gridDim.x) {
            const GroupedTile t = tile_at(slot);
            if (t.depth > 0) return t;
        }
        return GroupedTile{walk.all, -1, 0, 0, 0, 0, 0, 0};
    };
    // the tiles of groups without rows
    if (MODE == Grouped::TN && !p.accumulate)
        for (int slot = blockIdx.x; slot < slots; slot += gridDim.x) {
            const GroupedTile t = tile_at(slot);
            if (t.group < 0 || t.depth > 0) continue;
            for (int r = wave; r < t.rows; r += 4) {
                float* const line = static_cast<float*>(p.out) + (size_t(t.group) * p.m + t.m0 + r) * p.n + t.n0;
                for (int c = 4 * lane; c < t.cols; c += 4 * kWaveSize) *reinterpret_cast<f32x4*>(line + c) = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    GroupedTile cur = seek(blockIdx.x);
    if (cur.depth == 0) return;

    // Four consecutive passes of a wave's copies share one LDS base (M0) and differ in the instruction's immediate offset, which the hardware adds on the LDS side and on
    // the global side alike: the lane offsets take it back out, and the descriptors start kCopyBias bytes early so that no lane offset goes below zero.
    const uint32_t ld_a = uint32_t(MODE == Grouped::TN ? p.m : p.k) * 2, ld_b = uint32_t(MODE == Grouped::NT ? p.k : p.n) * 2;
    auto describe = [&](const uint8_t* base, long long bytes) __attribute__((always_inline)) { return make_rsrc(base - kCopyBias, biased_reach(bytes)); };
    // A plain operand's pass r of wave w has rows 128 (r / 4) + 32 w + 8 (r % 4) .. + 7, a turned one's k 16 w + 2 r and the one behind. `l`: the lane, out of which all of
    // this is worked out anew where it is needed, since the registers are.
    auto plain_row = [&](int l, int r) __attribute__((always_inline)) { return 128 * (r / 4) + 32 * wave + 8 * (r % 4) + (l >> 3); };
    auto plain_chunk = [&](int l, int r) __attribute__((always_inline)) { return (l & 7) ^ (l >> 3) ^ (r & 1); };
    auto turned_row = [&](int l, int r) __attribute__((always_inline)) { return 16 * wave + 2 * r + l / 32; };
    auto turned_chunk = [&](int l, int r, int columns) __attribute__((always_inline)) { return min((l & 31) ^ (Turned<BLOCK>::spread(turned_row(l, r)) << 1), columns / 8 - 1); };
    auto unit_base = [&](int r, bool turned) __attribute__((always_inline)) { return turned ? wave * 8192 + (r / 4) * 4096 : (r / 4) * 16384 + wave * 4096; };
    auto lane_anew = [&] __attribute__((always_inline)) {
        int l = lane;
        asm volatile("" : "+v"(l));
        return l;
    };
    auto product = [](uint32_t row, uint32_t ld, uint32_t more) __attribute__((always_inline)) {
        uint32_t v = row * ld + more;
        asm volatile("" : "+v"(v));         // (else it keeps the upper half of a 64-bit product's register pair)
        return v;
    };

    // Where the copies are: k-tile copy_kt of `ahead`, their operands' descriptors and lane offsets.
    GroupedTile ahead = cur;
    int copy_kt = 0;
    __amdgpu_buffer_rsrc_t rsrc_a, rsrc_b;
    uint32_t voff_a[8], voff_b[8];
    const uint8_t *from_a, *from_b;         // of turned operands: where the k-tile starts
    // SOURCES, a bit a pass: the gathered row that this lane copies is none. Eight of the copies' k-tile, behind them eight each of the one before and of that before it.
    uint32_t none_of = 0;
    auto age_none = [&] __attribute__((always_inline)) { if (SOURCES) none_of = (none_of & 0xff) | none_of << 8; };
    i32x16_unaligned sources;               // SOURCES: of this wave's rows of the k-tile
    auto here_of = [&](const GroupedTile& t, int kt) __attribute__((always_inline)) { return min(kDepth, t.depth - kt * kDepth); };
    // The lane offsets, of turned operands for k-tiles of which `here` of k are copied. They are the same for all tiles that are whole, and so is what they were last worked out for.
    // What is copied of k behind the contraction's end is made zeros later; it only has to exist, and so it does, as the next row's or as rows of another group, but at the end of a
    // turned operand: there the last k-tile (`tail_aims`) has its own last row instead. Of a plain operand's last row that is out of the descriptor's range, for some lanes of a copy.
    bool aimed_whole = false, tail_aims = false;
    auto aim_lanes = [&](int here) __attribute__((always_inline)) {
        const GroupedTile& t = ahead;
        const bool whole = !GATHER_A && here == kDepth && t.rows == BLOCK && t.cols == BLOCK;
        if (whole && aimed_whole) return;
        aimed_whole = whole;
        const int l = lane_anew();
#pragma unroll
        for (int r = 0; r < PASSES; ++r) {
            const uint32_t bias = kCopyBias - (r % 4) * 1024, in_row = plain_chunk(l, r) * kChunk + bias;
            if constexpr (TURN_A) {
                voff_a[r] = product(min(turned_row(l, r), here - 1), ld_a, turned_chunk(l, r, t.rows) * kChunk + bias);
            } else {
                int row = min(plain_row(l, r), t.rows - 1);
                if constexpr (GATHER_A) {
                    const int s = p.source[t.m0 + row];
                    row = uint32_t(s) < uint32_t(p.source_rows) ? s : 0;
                }
                voff_a[r] = product(row, ld_a, in_row);
            }
            if constexpr (SOURCES) voff_b[r] = turned_chunk(l, r, t.cols) * kChunk + bias;         // its row is added when it is known
            else if constexpr (TURN_B) voff_b[r] = product(min(turned_row(l, r), here - 1), ld_b, turned_chunk(l, r, t.cols) * kChunk + bias);
            else voff_b[r] = product(min(plain_row(l, r), t.cols - 1), ld_b, in_row);
        }
    };
    auto describe_turned = [&] __attribute__((always_inline)) {
        const GroupedTile& t = ahead;
        const int row = t.k0 + copy_kt * kDepth;
        if constexpr (TURN_A) rsrc_a = describe(from_a, (long long)(p.rows - row) * ld_a - t.m0 * 2);
        if constexpr (MODE == Grouped::TN && !SOURCES) rsrc_b = describe(from_b, (long long)(p.rows - row) * ld_b - t.n0 * 2);
        if constexpr (MODE == Grouped::NN) rsrc_b = describe(from_b, ((long long)(p.groups - t.group) * p.k - row) * ld_b - t.n0 * 2);
    };
    auto aim_copies = [&] __attribute__((always_inline)) {
        const GroupedTile& t = ahead;
        if constexpr (TURN_A) from_a = p.lhs + size_t(t.k0) * ld_a + t.m0 * 2;
        else if constexpr (GATHER_A) rsrc_a = describe(p.lhs, (long long)p.source_rows * ld_a);
        else rsrc_a = describe(p.lhs + size_t(t.m0) * ld_a, (long long)t.rows * ld_a);
        const uint8_t* const rhs = MODE == Grouped::TN ? p.rhs : p.rhs + size_t(t.group) * p.n * p.k * 2;
        if constexpr (SOURCES) rsrc_b = describe(p.rhs + t.n0 * 2, (long long)p.source_rows * ld_b - t.n0 * 2);
        else if constexpr (TURN_B) from_b = rhs + size_t(t.k0) * ld_b + t.n0 * 2;
        else rsrc_b = describe(rhs + size_t(t.n0) * ld_b, (long long)t.cols * ld_b);
        describe_turned();
        tail_aims = t.depth % kDepth != 0 && (MODE == Grouped::TN ? t.k0 + t.count() * kDepth > p.rows : MODE == Grouped::NN && weights_end_inside(p.groups - t.group, p.k));
        aim_lanes(tail_aims ? here_of(t, 0) : kDepth);
    };
    // Behind the walk's last k-tile that one is copied again, two times, into units that nobody reads any more: the count of copies under way stays what the waits below take it for.
    bool walking = true;
    // the tiles behind the current one, as far as the copies have come: up to three, of one k-tile each; and how many k of the next one's first k-tile exist
    int next1 = 0, next2 = 0, next3 = 0, lead = 0, next_here = kDepth;
    // Most k-tiles are followed by a whole one of the same tile: what that takes is a few scalar instructions, which ride under the last MFMAs of a k-tile.
    auto within = [&] __attribute__((always_inline)) { return (copy_kt + 1) * kDepth + (tail_aims ? kDepth : 1) <= ahead.depth; };
    auto advance_within = [&] __attribute__((always_inline)) {
        ++copy_kt;
        if constexpr (TURN_A) from_a += size_t(kDepth) * ld_a;
        if constexpr (TURN_B && !SOURCES) from_b += size_t(kDepth) * ld_b;
        describe_turned();
    };
    auto advance_beyond = [&] __attribute__((always_inline)) {
        if (!walking) return;
        if (copy_kt + 1 < ahead.count()) {          // a last k-tile that is aimed at anew
            advance_within();
            aim_lanes(here_of(ahead, copy_kt));
            return;
        }
        const GroupedTile next = seek(ahead.slot + gridDim.x);
        walking = next.depth != 0;
        if (!walking) return;
        ahead = next, copy_kt = 0;
        const int waiting = next.packed(lane);
        next1 = lead == 0 ? waiting : next1, next2 = lead == 1 ? waiting : next2, next3 = lead == 2 ? waiting : next3;
        next_here = lead == 0 ? here_of(next, 0) : next_here;
        ++lead;
        aim_copies();
    };
    // the sources of this wave's 16 rows of the copies' k-tile
    auto load_sources = [&] __attribute__((always_inline)) {
        if constexpr (SOURCES) {
            typedef const __attribute__((address_space(4))) int* Scalars;
            const Scalars from = (Scalars)(uintptr_t)(p.source + ahead.k0);
            const int first = copy_kt * kDepth + 16 * wave;
            if (first + 16 <= ahead.depth) {
                sources = *(const __attribute__((address_space(4))) i32x16_unaligned*)(from + first);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) sources[i] = from[min(first + i, ahead.depth - 1)];
            }
            none_of &= ~0xffu;
        }
    };
    auto copy = [&](__amdgpu_buffer_rsrc_t rsrc, uint32_t voff, uint32_t at, int r, int base) __attribute__((always_inline)) {
        auto* to = YAN_LDS_PTR(ring + base);
        switch (r & 3) {        // the immediate offset is part of the instruction
            case 0: __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, kChunk, voff, at, 0 * 1024, 0); break;
            case 1: __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, kChunk, voff, at, 1 * 1024, 0); break;
            case 2: __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, kChunk, voff, at, 2 * 1024, 0); break;
            default: __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, kChunk, voff, at, 3 * 1024, 0); break;
        }
    };
    auto copy_a = [&](int r, int unit) __attribute__((always_inline)) {
        copy(rsrc_a, voff_a[r], TURN_A ? 0u : uint32_t(copy_kt) * kRowBytes, r, unit + unit_base(r, TURN_A));
    };
    auto copy_b = [&](int r, int unit) __attribute__((always_inline)) {
        uint32_t voff = voff_b[r];
        if constexpr (SOURCES) {
            const int s0 = sources[2 * r], s1 = sources[2 * r + 1];
            const bool there0 = uint32_t(s0) < uint32_t(p.source_rows), there1 = uint32_t(s1) < uint32_t(p.source_rows);
            const uint32_t at0 = there0 ? uint32_t(s0) * ld_b : 0u, at1 = there1 ? uint32_t(s1) * ld_b : 0u;
            voff += lane < 32 ? at0 : at1;
            none_of |= (lane < 32 ? there0 : there1) ? 0u : 1u << r;
        }
        copy(rsrc_b, voff, TURN_B ? 0u : uint32_t(copy_kt) * kRowBytes, r, unit + unit_base(r, TURN_B));
    };
    // Zeros in place of what the k-tile in units (a, b) has been given for what does not exist, by the wave that copied it, `age` k-tiles before the last one that it did.
    auto clear = [&](int here, int age, int a, int b) __attribute__((always_inline)) {
        // (of turned operands a wave has copied 16 k)
        const bool none_of_mine = TURN_A && TURN_B ? 16 * wave + 16 <= here : here == kDepth;
        const uint32_t none_here = none_of >> (8 * age) & 0xff;
        if (none_of_mine && !(SOURCES && __ballot(none_here != 0))) return;
        const i32x4 zeros = i32x4{0, 0, 0, 0};
        const int l = lane_anew();
#pragma unroll
        for (int r = 0; r < PASSES; ++r) {
            const int place = (r & 3) * 1024 + l * kChunk;
            // (of a row without a source both operands, which have the same rows in the same lanes: it counts for nothing, whatever the other has there)
            const bool plain_tail = plain_chunk(l, r) >= here / 8, turned_tail = turned_row(l, r) >= here || (SOURCES && ((none_here >> r) & 1));
            if (TURN_A ? turned_tail : plain_tail) *reinterpret_cast<i32x4*>(ring + a + unit_base(r, TURN_A) + place) = zeros;
            if (TURN_B ? turned_tail : plain_tail) *reinterpret_cast<i32x4*>(ring + b + unit_base(r, TURN_B) + place) = zeros;
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoWaitVm, 0));
    };

    f32x4 acc[TN][TM];
    Frag nf[2][TN], mf[2][TM];
    auto mma = [&](auto first_c, auto kh_c, int i, int j) __attribute__((always_inline)) {
        constexpr int KH = decltype(kh_c)::value;
        f32x4& sum = acc[i][j];
        const Frag &n = nf[KH][i], &m = mf[KH][j];
        if constexpr (decltype(first_c)::value) {
            if constexpr (__is_same(Elem, __bf16)) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=a"(sum) : "v"(n), "v"(m));
            else asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, 0" : "=a"(sum) : "v"(n), "v"(m));
        } else {
            if constexpr (__is_same(Elem, __bf16)) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(sum) : "v"(n), "v"(m));
            else asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(sum) : "v"(n), "v"(m));
        }
    };
    const int plain[2] = {frag_offset<16>(lane, 2 * g), frag_offset<16>(lane, 2 * g + 1)}, turned = Turned<BLOCK>::lane_offset(lane);
    // fragment j of the rows, i of the columns, of half RK of the k-tile in unit `unit`; a turned one in two reads, of which this is number `part`
    auto read_m = [&](auto kh_c, auto rk_c, int unit, int j, int part) __attribute__((always_inline)) {
        constexpr int KH = decltype(kh_c)::value, RK = decltype(rk_c)::value;
        if constexpr (TURN_A) read_turned_part<Frag>(mf[KH][j], ring + unit + RK * 8 * ROW_BYTES + part * 4 * ROW_BYTES + (turned ^ ((2 * j + wm) * 32)), part);
        else mf[KH][j] = *reinterpret_cast<const Frag*>(ring + unit + (32 * j + 16 * wm) * kRowBytes + plain[RK]);
    };
    auto read_n = [&](auto kh_c, auto rk_c, int unit, int i, int part) __attribute__((always_inline)) {
        constexpr int KH = decltype(kh_c)::value, RK = decltype(rk_c)::value;
        if constexpr (TURN_B) read_turned_part<Frag>(nf[KH][i], ring + unit + RK * 8 * ROW_BYTES + part * 4 * ROW_BYTES + (turned ^ ((8 * wn + i) * 32)), part);
        else nf[KH][i] = *reinterpret_cast<const Frag*>(ring + unit + (128 * wn + 16 * i) * kRowBytes + plain[RK]);
    };
    constexpr int PARTS_A = TURN_A ? 2 : 1, PARTS_B = TURN_B ? 2 : 1;
    using Half0 = std::integral_constant<int, 0>;
    using Half1 = std::integral_constant<int, 1>;
    // read number x of a half's fragments, those of the rows first; `whole`: of all eight row atoms, or of four
    auto read = [&](auto kh_c, auto rk_c, auto tm_c, int a, int b, int x) __attribute__((always_inline)) {
        constexpr int RM = decltype(tm_c)::value * PARTS_A;
        if (x < RM) read_m(kh_c, rk_c, a, x / PARTS_A, x % PARTS_A);
        else if (x - RM < TN * PARTS_B) read_n(kh_c, rk_c, b, (x - RM) / PARTS_B, (x - RM) % PARTS_B);
    };
    // Half a k-tile: TN rows of TMR MFMAs on fragment buffer KH. Beside all rows but the last one go COPIES copies and the reads of the next half (units a, b; half RK) into the
    // other buffer, beside the last one what `last_row(j)` does, j = 0 .. TMR - 1. The next half may be another tile's, with all of its row atoms: those are always read.
    auto half_step = [&](auto kh_c, auto rk_c, auto first_c, auto tm_c, auto copies_c, int a, int b, auto&& copy_one, auto&& last_row) __attribute__((always_inline)) {
        constexpr int KH = decltype(kh_c)::value, TMR = decltype(tm_c)::value, COPIES = decltype(copies_c)::value;
        using Other = std::integral_constant<int, KH ^ 1>;
        using ReadM = std::integral_constant<int, TM>;
        constexpr int ALL = TM * PARTS_A + TN * PARTS_B, SIDE = ALL + COPIES, SLOTS = (TN - 1) * TMR;
        static_for<TN * TMR>([&](auto slot_c) __attribute__((always_inline)) {
            constexpr int SLOT = decltype(slot_c)::value;
            mma(first_c, kh_c, SLOT / TMR, SLOT % TMR);
            if constexpr (SLOT >= SLOTS) {
                last_row(SLOT - SLOTS);
            } else {
                // copies and reads evenly among each other and over the MFMAs
                constexpr int FROM = SLOT * SIDE / SLOTS, UPTO = (SLOT + 1) * SIDE / SLOTS;
                static_for<UPTO - FROM>([&](auto s_c) __attribute__((always_inline)) {
                    constexpr int S = FROM + decltype(s_c)::value, COPIED = S * COPIES / SIDE;
                    if constexpr ((S + 1) * COPIES / SIDE > COPIED) copy_one(COPIED);
                    else read(Other{}, rk_c, ReadM{}, a, b, S - COPIED);
                });
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto meet = [] __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // the first two k-tiles of the walk into units 0 .. 3
    aim_copies();
    for (int s = 0; s < 2; ++s) {
        load_sources();
#pragma unroll
        for (int r = 0; r < PASSES; ++r) copy_a(r, 2 * s * UNIT_BYTES);
#pragma unroll
        for (int r = 0; r < PASSES; ++r) copy_b(r, (2 * s + 1) * UNIT_BYTES);
        age_none();
        if (within()) advance_within();
        else advance_beyond();
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
    asm volatile("" ::: "memory");
    clear(here_of(cur, 0), 2, 0, UNIT_BYTES);
    meet();
#pragma unroll
    for (int x = 0; x < TM * PARTS_A + TN * PARTS_B; ++x) read(Half0{}, Half0{}, std::integral_constant<int, TM>{}, 0, UNIT_BYTES, x);
    __builtin_amdgcn_sched_barrier(0);

    const bool stream_out = MODE == Grouped::TN ? size_t(p.groups) * p.m * p.n * 4 > (size_t(32) << 20) : size_t(p.m) * p.n * 2 > (size_t(32) << 20);
    // stores of a tile by a wave, whatever of it exists, and how many of them are behind the current tile's first copies
    constexpr int STORES_ALL = MODE == Grouped::TN ? 64 : 32;
    int stores_before = 0;
    auto wait_for_all_but = [](auto count_c) __attribute__((always_inline)) {
        constexpr int MOST = decltype(count_c)::value < kNoWaitVm ? decltype(count_c)::value : kNoWaitVm;
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(MOST, 0));
    };
    // byte offsets of the units that hold A and B of the current k-tile, of the next one, and of the fifth unit
    int oa = 0, ob = UNIT_BYTES, oa1 = 2 * UNIT_BYTES, ob1 = 3 * UNIT_BYTES, o5 = 4 * UNIT_BYTES;
    while (true) {
        const int count = cur.count();
        using AllCopies = std::integral_constant<int, PASSES>;
        auto nothing = [](int) __attribute__((always_inline)) {};
        auto k_tile = [&](auto first_c, auto tm_c, int kt) __attribute__((always_inline)) {
            load_sources();
            // (a tile of up to 128 rows has no second half of rows to copy, but for columns in a turned operand's rows, which come with the others')
            int passes = __builtin_amdgcn_readfirstlane(TURN_A || ahead.rows > 128 ? PASSES : PASSES / 2);
            asm volatile("" : "+s"(passes));            // (a number, of which every copy is one compare)
            half_step(Half0{}, Half1{}, first_c, tm_c, AllCopies{}, oa, ob,
                      [&](int r) __attribute__((always_inline)) { if (TURN_A || r < PASSES / 2 || passes == PASSES) copy_a(r, o5); }, nothing);
            // The next k-tile has landed. Behind its copies a wave has issued those above and, in a tile's first k-tile, the stores of the tile before; neither need be done.
            if constexpr (decltype(first_c)::value) {
                if (stores_before == STORES_ALL) wait_for_all_but(std::integral_constant<int, STORES_ALL + PASSES / 2>{});
                else if (stores_before == STORES_ALL * 3 / 4) wait_for_all_but(std::integral_constant<int, STORES_ALL * 3 / 4 + PASSES / 2>{});
                else if (stores_before == STORES_ALL / 2) wait_for_all_but(std::integral_constant<int, STORES_ALL / 2 + PASSES / 2>{});
                else if (stores_before == STORES_ALL / 4) wait_for_all_but(std::integral_constant<int, STORES_ALL / 4 + PASSES / 2>{});
                else wait_for_all_but(std::integral_constant<int, PASSES / 2>{});
            } else {
                wait_for_all_but(std::integral_constant<int, PASSES>{});
                if (!TURN_A && passes != PASSES) wait_for_all_but(std::integral_constant<int, PASSES / 2>{});
            }
            asm volatile("" ::: "memory");
            if (SOURCES || kt + 2 >= count) clear(kt + 1 == count ? next_here : here_of(cur, kt + 1), 1, oa1, ob1);
            meet();                             // every wave is done reading this k-tile
            const int into = oa;
            bool inside;
            half_step(Half1{}, Half0{}, std::false_type{}, tm_c, AllCopies{}, oa1, ob1, [&](int r) __attribute__((always_inline)) { copy_b(r, into); },
                      [&](int j) __attribute__((always_inline)) {
                          if (j == 0) inside = within();
                          if (j == 1) age_none();
                          if (j == 1) { const int ta = oa1; oa1 = o5; o5 = ob; ob = ob1; ob1 = oa; oa = ta; }
                          if (j == (decltype(tm_c)::value > 2 ? 2 : 1) && inside) advance_within();
                      });
            if (!inside) advance_beyond();
        };
        auto walk_k = [&](auto tm_c) __attribute__((always_inline)) {
            k_tile(std::true_type{}, tm_c, 0);
            for (int kt = 1; kt < count; ++kt) k_tile(std::false_type{}, tm_c, kt);
        };
        // The 4 registers of atom (i, j) are columns 128 wn + 16 i + 4 g + {0..3} of row 32 j + 16 wm + col. Each wave turns its slab round through the fifth unit, 16 rows by 64
        // columns at a time and two such pieces in turn: the sums of piece u go in, piece u - 1 comes out, piece u - 2 is stored.
        uint32_t gone = 0;                      // GATHER_A, a bit an atom of rows: this lane's row in it has no source, and its outputs are zeros whatever the weights hold
        auto epilogue = [&](auto policy_c, auto tm_c, auto accumulate_c) __attribute__((always_inline)) {
            constexpr bool ACCUMULATE = decltype(accumulate_c)::value, WIDE = MODE == Grouped::TN;          // fp32 outputs
            constexpr int SIZE = WIDE ? 4 : 2, PIECE = 64, PITCH = WIDE ? PIECE * 4 : PIECE * 2 + 16, PIECE_BYTES = 16 * PITCH, PIECES = 2 * decltype(tm_c)::value;
            constexpr int LANES_PER_ROW = PIECE * SIZE / 16, ROWS_PER_STORE = kWaveSize / LANES_PER_ROW, STORES = 16 / ROWS_PER_STORE, AHEAD = 1;
            static_assert(PIECES * STORES == STORES_ALL * decltype(tm_c)::value / TM);
            static_assert(4 * 2 * PIECE_BYTES <= UNIT_BYTES);
            uint8_t* const buffers = ring + o5 + wave * (2 * PIECE_BYTES);
            const uint32_t row_bytes = uint32_t(p.n) * SIZE;
            const size_t first = WIDE ? (size_t(cur.group) * p.m + cur.m0) * p.n + cur.n0 : size_t(cur.m0) * p.n + cur.n0;
            const __amdgpu_buffer_rsrc_t rsrc_out = make_rsrc(static_cast<uint8_t*>(p.out) + first * SIZE, uint32_t(cur.rows) * row_bytes - uint32_t(cur.n0) * SIZE);
            const int row_in = lane / LANES_PER_ROW, c = lane % LANES_PER_ROW;
            // chunk c of a row of fp32 in slot c ^ row; rows of 16 bits 16 bytes further apart than they are long
            const auto place = [&](int row, int chunk) __attribute__((always_inline)) { return row * PITCH + (WIDE ? (chunk ^ (row & (LANES_PER_ROW - 1))) : chunk) * 16; };
            uint32_t off[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int column = 128 * wn + PIECE * h + c * (16 / SIZE);
                off[h] = column < cur.cols ? uint32_t(16 * wm + row_in) * row_bytes + uint32_t(column) * SIZE : kOutOfRange;
            }
            [[maybe_unused]] const bool any_gone = __ballot(gone != 0) != 0;
            i32x4 back[2][STORES], held[ACCUMULATE ? AHEAD + 1 : 1][STORES];
            auto load = [&](int u) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < STORES; ++s) {
                    uint32_t down = uint32_t(u / 2 * 32 + ROWS_PER_STORE * s) * row_bytes;
                    asm volatile("" : "+s"(down));          // (added here, not ahead of the walk into a register for each)
                    held[u % (AHEAD + 1)][s] = __builtin_amdgcn_raw_buffer_load_b128(rsrc_out, off[u % 2] + down, 0, 0);
                }
            };
            if constexpr (ACCUMULATE) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) load(u);
            }
#pragma unroll
            for (int u = 0; u < PIECES + 2; ++u) {
                if (u < PIECES) {
                    const int j = u / 2, h = u % 2;
#pragma unroll
                    for (int a = 0; a < PIECE / 16; ++a) {
                        // the sums come out of the accumulation registers here and nowhere earlier
                        const f32x4& sum = acc[h * (PIECE / 16) + a][j];
                        f32x4 v;
                        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[0]) : "a"(sum[0]));
                        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[1]) : "a"(sum[1]));
                        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[2]) : "a"(sum[2]));
                        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[3]) : "a"(sum[3]));
                        if constexpr (GATHER_A) {
                            if (any_gone) v = (gone >> j) & 1 ? f32x4{0.f, 0.f, 0.f, 0.f} : v;
                        }
                        uint8_t* const to = buffers + (u & 1) * PIECE_BYTES;
                        if constexpr (WIDE) *reinterpret_cast<f32x4*>(to + place(col, 4 * a + g)) = v;
                        else *reinterpret_cast<decltype(pack4(v, Elem{}))*>(to + place(col, 0) + (16 * a + 4 * g) * 2) = pack4(v, Elem{});
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                if (u >= 1 && u - 1 < PIECES) {
#pragma unroll
                    for (int s = 0; s < STORES; ++s) back[(u - 1) & 1][s] = *reinterpret_cast<const i32x4*>(buffers + ((u - 1) & 1) * PIECE_BYTES + place(ROWS_PER_STORE * s + row_in, c));
                }
                if (u >= 2) {
                    const int w = u - 2;
                    if constexpr (ACCUMULATE) {
                        if (w + AHEAD < PIECES) load(w + AHEAD);
                    }
#pragma unroll
                    for (int s = 0; s < STORES; ++s) {
                        i32x4 v = back[w & 1][s];
                        if constexpr (ACCUMULATE) v = __builtin_bit_cast(i32x4, __builtin_bit_cast(f32x4, v) + __builtin_bit_cast(f32x4, held[w % (AHEAD + 1)][s]));
                        // (all of the offset in the lane's register, see wgrad_store in fp8_wgrad.hpp)
                        uint32_t down = uint32_t(w / 2 * 32 + ROWS_PER_STORE * s) * row_bytes;
                        if constexpr (WIDE) asm volatile("" : "+s"(down));
                        buffer_store_16(v, rsrc_out, off[w % 2] + down, decltype(policy_c)::value);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto leave = [&](auto tm_c, auto accumulate_c) __attribute__((always_inline)) {
            if (stream_out) epilogue(std::true_type{}, tm_c, accumulate_c);
            else epilogue(std::false_type{}, tm_c, accumulate_c);
        };
        auto tile = [&](auto tm_c) __attribute__((always_inline)) {
            walk_k(tm_c);
            if constexpr (GATHER_A) {
#pragma unroll
                for (int j = 0; j < decltype(tm_c)::value; ++j) {
                    const int s = p.source[cur.m0 + min(32 * j + 16 * wm + col, cur.rows - 1)];
                    gone |= uint32_t(s) < uint32_t(p.source_rows) ? 0u : 1u << j;
                }
            }
            asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");      // the last MFMAs retire before the sums are read
            if (MODE == Grouped::TN && p.accumulate) leave(tm_c, std::bool_constant<MODE == Grouped::TN>{});
            else leave(tm_c, std::false_type{});
        };
        // (both branches to the end of the tile: sums that a flat tile does not have would else be kept for it)
        if (MODE != Grouped::TN && cur.rows <= 64) tile(std::integral_constant<int, TM / 4>{});
        else if (cur.rows <= 128) tile(std::integral_constant<int, TM / 2>{});
        else if (MODE != Grouped::TN && cur.rows <= 192) tile(std::integral_constant<int, TM * 3 / 4>{});
        else tile(std::integral_constant<int, TM>{});
        if (lead == 0) break;
        stores_before = MODE == Grouped::TN ? ceil_div(cur.rows, 128) * (STORES_ALL / 2) : ceil_div(cur.rows, 64) * (STORES_ALL / 4);
        cur = GroupedTile::unpacked(next1);
        next1 = next2, next2 = next3;
        --lead;
        next_here = lead ? here_of(GroupedTile::unpacked(next1), 0) : kDepth;
        // every wave is out of the fifth unit before the next copies go into it
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoWaitVm, 0));
        meet();
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));          // the copies behind the last k-tile have landed: the LDS may be another's from here on
}

enum Grouped16Kernel { kGroupedAny, kGroupedTall, kGrouped128, kGrouped64, kGrouped32 };

// The kernel for a product: by the rows of a group on average, and by how many tiles of a kind there are at most for the chip's compute units. How the rows are spread over the groups is
// on the device, where the host cannot look: a few long groups among many short ones go by the mean of them all, and may get smaller tiles than they would alone. Fitted to every kernel's time
// over 4 to 256 groups of 2 to 640 rows, (n, k) of 1024 x 512, 2048 x 2048, 4096 x 7168 and 7168 x 2048, bf16, on 256 compute units; over these the choice is 1.7 % (NT, NN)
// and 0.5 % (TN) behind the best of the kernels in the mean, and 26 % at worst (16 groups of 24 rows, 7168 x 2048: 113, with 32 x 128 tiles 89). Microseconds, NT unless it says TN:
//   256 x 256 tiles: one workgroup a compute unit, so the tiles have to number nearly as many. 16 groups of 81 rows, 4096 x 7168: 178 with them, 259 with 128 x 128. 64 groups of 88 rows,
//       2048 x 2048: 130 | 141. Long groups earn them with fewer tiles: 4 of 496 rows, 4096 x 7168 (176 tiles): 128 | 180. Not so 4 of 522 rows, 1024 x 512 (48 tiles): 13.0 | 9.9.
//       TN: 16 groups of 113 rows, 4096 x 7168 (7168 tiles): 368 | 394, 64 of 190, 1024 x 512 (512 tiles): 34 | 42, but 4 of 116, 7168 x 2048 (896 tiles): 64 | 52: few rows make a tile's
//       stores most of its work, and two workgroups a compute unit overlap one's with the other's loads.
//   32 x 128 tiles: up to 16 rows a group, few of which pass 32 then: 256 groups of 1 row, 1024 x 512: 47.6 with them, 62.4 with 64 x 64. 16 groups of 23 rows, 2048 x 2048: 30.1 | 23.0.
//   64 x 64 tiles for as long as they come to about one round of two workgroups a compute unit: 4 groups of 26 rows, 4096 x 7168 (320 tiles): 37.5 with them, 74 with 128 x 128. 4 of 207
//       rows, 2048 x 2048 (544): 16.6 | 25.4. 16 of 122 rows, 1024 x 512 (624): 12.2 | 10.1. 64 of 63 rows, 7168 x 2048 (14112): 488 | 356. TN, 4 groups, 1024 x 512 (512): 11.5 | 14.6.
template <Grouped MODE>
inline Grouped16Kernel grouped16_plan(int groups, int rows, int m, int n, int k, int cus) {
    const int each = rows / groups;
    const auto tiles = [&](int block_m, int block_n) {
        return (MODE == Grouped::TN ? (long long)groups * ceil_div(m, block_m) : (long long)most_row_tiles(rows, groups, block_m)) * ceil_div(n, block_n);
    };
    if (MODE == Grouped::TN) {
        if ((each >= 80 && tiles(256, 256) >= cus * 6ll) || (each >= 160 && tiles(256, 256) * 4 >= cus * 5ll)) return kGroupedTall;
        return tiles(128, 128) * 4 >= cus * 3ll ? kGrouped128 : kGrouped64;
    }
    if (k != 0 && ((each >= 80 && tiles(256, 256) * 8 >= cus * 7ll) || (each >= 192 && tiles(256, 256) * 8 >= cus * 5ll))) return kGroupedTall;
    if (each <= 16) return kGrouped32;
    return tiles(64, 64) * 3 >= cus * 7ll ? kGrouped128 : kGrouped64;
}

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
        return ceil_div<long long>((long long)most_row_tiles(m, groups, block_m) * ceil_div(n, block_n), kNumXCD) * kNumXCD;
    };
    const auto launch = [&](auto kernel, int block_m, int block_n) {
        const long long slots = slots_of(block_m, block_n);
        if (slots >= 1ll << 30) return hipErrorInvalidValue;
        const int most = int(std::min(slots, 1ll << 20));             // a launch has less than 2^32 threads: beyond this a workgroup has several tiles
        hipLaunchKernelGGL(kernel, dim3(uint32_t(capped ? capped_grid(most, num_sms, device_cu_count()) : most)), dim3(256), 0, stream, p, int(slots));
        return hipGetLastError();
    };
    const Grouped16Kernel which = KERNEL != kGroupedAny ? KERNEL : grouped16_plan<MODE>(groups, rows, m, n, k, device_cu_count());
    switch (which) {
        case kGroupedTall: {
            if (MODE != Grouped::TN && k == 0) return hipErrorInvalidValue;
            const int cus = capped ? capped_grid(device_cu_count(), num_sms, device_cu_count()) : device_cu_count() / kNumXCD * kNumXCD;
            const long long slots = MODE == Grouped::TN ? ceil_div<long long>((long long)groups * ceil_div(m, 256) * ceil_div(n, 256), kNumXCD) * kNumXCD : slots_of(256, 256);
            if (slots >= 1ll << 30) return hipErrorInvalidValue;
            hipLaunchKernelGGL((grouped16_tall_kernel<Elem, MODE, GATHER>), dim3(uint32_t(std::min<long long>(cus, MODE == Grouped::TN ? slots : 2 * slots))), dim3(256), 0, stream, p);
            return hipGetLastError();
        }
        case kGrouped32:
            if constexpr (MODE != Grouped::TN) return launch(grouped16_kernel<Elem, MODE, 32, 128, 4, GATHER>, 32, 128);
            else return hipErrorInvalidValue;
        case kGrouped64: return launch(grouped16_kernel<Elem, MODE, 64, 64, 4, GATHER>, 64, 64);
        default: return launch(grouped16_kernel<Elem, MODE, 128, 128, 2, GATHER>, 128, 128);
    }
}

} // namespace yan
