// out[i, j] (+)= sum_b 2^(sa[i, b] + sb[j, b] - 254) sum_{t < 128} a[i, 128 b + t] b[j, 128 b + t]      (e4m3 x e4m3 -> fp32)
//
// The product of a weight gradient: both operands quantised 1 x 128 along K, which is the tokens, with power-of-two scales, the sums
// in fp32 and added to what is in `out` if asked. Grouped: K is cut at `offsets` (multiples of 128, on the device) and group g has its own
// out[g], the gradient of one expert's weights.
//
// The codes are multiplied as bf16, which holds code * 2^e exactly: gfx950 converts two codes and applies a power of two in one instruction, so
// the scales cost nothing and the sums stay in the matrix core's accumulators from the first k-tile to the last. The FP8 MFMAs are twice as
// fast and add up less exactly than fp32 sums do: small products next to large ones lose bits inside of the instruction, whatever its shape
// and also from a zero accumulator, 1.5e-5 of the result's norm for normal operands and 4e-5 to 5e-5 where values spread more widely, at K = 128 as at 16384 (bf16:
// 1e-8 to 7e-8 and 2e-7 to 9e-7).
// A gradient that is summed up in fp32 over micro-batches is to keep what fp32 keeps.
//
// Tiles are staged as in the other GEMMs (tile_io.hpp): 128-byte rows, swizzled, HBM -> LDS directly, in a ring. A row's scale bytes lie
// along K, rows a multiple of 4 bytes apart, so a lane loads those of four k-tiles as a dword.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_fp8.h>

#include <algorithm>
#include <type_traits>

#include "utils.hpp"
#include "mfma_utils.hpp"
#include "scheduler.hpp"
#include "tile_io.hpp"

namespace yan {

struct WgradProblem {
    const uint8_t *a, *b, *sa, *sb;         // codes [m, k], [n, k]; scale bytes, rows ld_sa, ld_sb apart
    float* out;                             // [groups, m, n]
    const int* offsets;                     // [groups + 1], or null: one group, all of K
    int m, n, k, ld_sa, ld_sb, groups;
    bool accumulate;
};

// Sums of K parts and the counters of their arrival, a counter a wave of every tile.
struct WgradWorkspace {
    float* sums;
    unsigned* counters;
};

// K range of a group in k-tiles. Offsets are the caller's, on the device: whatever they hold, the range lies inside K.
__device__ __forceinline__ void wgrad_range(const WgradProblem& p, int group, int& lo, int& hi) {
    const int k_tiles = p.k / 128;
    lo = 0, hi = k_tiles;
    if (p.offsets) {
        lo = min(max(p.offsets[group], 0) / 128, k_tiles);
        hi = max(lo, min(max(p.offsets[group + 1], 0) / 128, k_tiles));
    }
}

// Copies of a tile's k-tiles into LDS, in TileStager's layout: an instruction has 8 rows, pass j of wave w the group j * NUM_WAVES + w. Of the rows behind the
// operand's last one those in its group are out of range and become zeros; in the place of a group that is wholly behind it another one's rows are copied once more,
// sums of which nobody stores. That way no copy is out of range for every lane. Such a copy waits for nothing in memory, and the kernels below use the LDS
// again, for the next tile's rows and for their sums: they are not to rest on its zeros being there by the time that the wave's counter has it as done.
template <int ROWS, int NUM_WAVES>
struct WgradStager {
    static_assert(ROWS % (8 * NUM_WAVES) == 0 && NUM_WAVES % 2 == 0);
    static constexpr int PASSES = ROWS / 8 / NUM_WAVES;
    uint32_t chunk_at;              // of this lane's chunk in a group
    // Of its chunks in the tile. (A scalar offset a pass is a choice, a product and two sums behind every copy, and a lone wave has no room for them in the shadow
    // of its MFMAs: 99 k-tiles of 2048 x 4096 on 256 x 128 tiles 179 us, 162 so. The bound is a plain number since with PASSES, or anything else that depends on
    // the template's arguments, the compiler leaves out the host side of a kernel that is launched.)
    uint32_t voff[8];
    static_assert(PASSES <= 8);

    // Which group of an operand with `rows` >= 1 rows in the tile is copied for `group`.
    __host__ __device__ __forceinline__ static int source_group(int group, int rows) { return group < (rows - 1) >> 3 ? group : (rows - 1) >> 3; }

    __device__ __forceinline__ void init(uint32_t ld_bytes, int wave, int lane) {
        const int sub = lane >> 3, slot = lane & 7;
        chunk_at = uint32_t(sub) * ld_bytes + (slot ^ sub ^ (wave & 1)) * kChunk;         // (slot ^ swizzle_of_row of the row that the place in LDS is for)
    }
    __device__ __forceinline__ void aim(int rows, uint32_t ld_bytes, int wave) {
#pragma unroll
        for (int j = 0; j < PASSES; ++j) voff[j] = chunk_at + uint32_t(source_group(j * NUM_WAVES + wave, rows) * 8) * ld_bytes;
    }
    __device__ __forceinline__ void issue_pass(__amdgpu_buffer_rsrc_t rsrc, uint8_t* lds_tile, int k_byte0, int wave, int j) const {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, YAN_LDS_PTR(lds_tile + (j * NUM_WAVES + wave) * 8 * kRowBytes), kChunk, voff[j], k_byte0, 0, 0);
    }
    __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t rsrc, uint8_t* lds_tile, int k_byte0, int wave) const {
#pragma unroll
        for (int j = 0; j < PASSES; ++j) issue_pass(rsrc, lds_tile, k_byte0, wave, j);
    }
};

// Eight codes times a power of two (a float, of which the exponent counts) as bf16.
__device__ __forceinline__ bf16x8 wgrad_decode(int lo, int hi, float scale) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(lo), scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(lo), scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(hi), scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(hi), scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The scale of a k-tile out of the dword that holds those of four: `shift` is 8 times its place.
__device__ __forceinline__ float wgrad_scale(int quad, int shift) { return __builtin_bit_cast(float, ((uint32_t(quad) >> shift) & 0xff) << 23); }

// Four sums to memory. All of the offset is in the lane's register: of a store of 16 bytes whose offset is partly in a scalar register the compiler
// thinks that its data may be overwritten by the next instruction. It may not: the second register of some lanes then held what came next.
__device__ __forceinline__ void wgrad_store(f32x4 v, __amdgpu_buffer_rsrc_t rsrc, uint32_t offset, bool streaming) {
    buffer_store_16(__builtin_bit_cast(i32x4, v), rsrc, offset, streaming);
}

// Where the `parts` parts of a tile's K range meet, wave by wave, as in the other GEMMs (meet_partials in tile_io.hpp) with their number known at run
// time: a wave leaves its sums, and the one that comes last adds up all parts in the order of their ranges. True for that one. Written and read
// at device scope: the parts run on different XCDs. The counters are zero before and after.
template <int NW, int TN, int TM>
__device__ __forceinline__ bool wgrad_meet(f32x4 (&acc)[TN][TM], const WgradWorkspace& w, int tile, int part, int parts, int wave, int lane) {
    constexpr int kDeviceScope = 16, VECS = TN * TM;
    constexpr uint32_t VEC_BYTES = kWaveSize * 16, WAVE_BYTES = VECS * VEC_BYTES, PART_BYTES = NW * WAVE_BYTES;
    const __amdgpu_buffer_rsrc_t sums = make_rsrc(w.sums + size_t(tile) * parts * (PART_BYTES / 4), uint32_t(parts) * PART_BYTES);
    const uint32_t at = uint32_t(wave) * WAVE_BYTES + lane * 16;
#pragma unroll
    for (int v = 0; v < VECS; ++v)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, acc[v / TM][v % TM]), sums, at + part * PART_BYTES + v * VEC_BYTES, 0, kDeviceScope);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, kNoWaitLgkm));            // the sums have reached memory before the count is taken
    asm volatile("" ::: "memory");
    unsigned before = 0;
    unsigned* const counter = w.counters + tile * NW + wave;
    if (lane == 0) before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    before = __builtin_amdgcn_readfirstlane(before);
    asm volatile("" ::: "memory");
    if (before != unsigned(parts) - 1) return false;
#pragma unroll
    for (int v = 0; v < VECS; ++v) acc[v / TM][v % TM] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int TOGETHER = 8;             // parts whose loads are under way at once
    for (int s0 = 0; s0 < parts; s0 += TOGETHER) {
        i32x4 raw[TOGETHER][VECS];
#pragma unroll
        for (int s = 0; s < TOGETHER; ++s)
#pragma unroll
            for (int v = 0; v < VECS; ++v)          // (past the last part: out of range, zeros)
                raw[s][v] = __builtin_amdgcn_raw_buffer_load_b128(sums, s0 + s < parts ? at + (s0 + s) * PART_BYTES + v * VEC_BYTES : kOutOfRange, 0, kDeviceScope);
#pragma unroll
        for (int s = 0; s < TOGETHER; ++s)
#pragma unroll
            for (int v = 0; v < VECS; ++v) acc[v / TM][v % TM] += __builtin_bit_cast(f32x4, raw[s][v]);
    }
    if (lane == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

// The smaller tiles: 4 waves, up to two workgroups a compute unit, which hide each other's waits; one tile a workgroup, or a walk under a cap. SPLIT: a slot
// is one of `parts` parts of a tile's K range.
template <int BLOCK_M, int BLOCK_N, int STAGES, bool SPLIT>
__global__ void __launch_bounds__(256, 2)
fp8_wgrad_kernel(WgradProblem p, WgradWorkspace w, int parts) {
    constexpr int NW = 4, WTM = BLOCK_M / 2, WTN = BLOCK_N / 2, TM = WTM / 16, TN = WTN / 16;
    using StA = WgradStager<BLOCK_M, NW>;
    using StB = WgradStager<BLOCK_N, NW>;
    constexpr int NUM_COPIES = StA::PASSES + StB::PASSES + 1, A_BYTES = BLOCK_M * kRowBytes, STAGE_BYTES = (BLOCK_M + BLOCK_N) * kRowBytes;
    static_assert((STAGES - 1) * NUM_COPIES <= 63);
    // Scales are copied with their k-tile, a dword of four k-tiles' a row, a row a lane: loaded into registers every fourth k-tile they made the wave wait for all
    // copies under way (64 tiles of 64 x 64, 64 k-tiles: 54.7 us, 36.5 so; 512 of 128 x 128, 64 k-tiles: 87.5 / 82.2).
    constexpr int SCALE_ROWS = NW * kWaveSize;
    static_assert(BLOCK_M % kWaveSize == 0 && BLOCK_M + BLOCK_N <= SCALE_ROWS);
    __shared__ __attribute__((aligned(1024))) uint8_t ring[STAGES * STAGE_BYTES];
    __shared__ __attribute__((aligned(1024))) uint32_t ring_scales[STAGES * SCALE_ROWS];

    const XcdTileScheduler<> sched(p.m, p.n, BLOCK_M, BLOCK_N);
    const int per_group = sched.grid_size(), slots = per_group * p.groups * (SPLIT ? parts : 1);
    const int lane = get_lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int wn = wave % 2, wm = wave / 2, g = lane / 16, col = lane % 16;
    for (int slot = blockIdx.x; slot < slots; slot += gridDim.x) {
        // the parts of a tile are neighbouring slots
        const int part = SPLIT ? slot % parts : 0, tile_slot = SPLIT ? slot / parts : slot, group = tile_slot / per_group;
        const TileCoord tile = sched.tile_of(tile_slot - group * per_group);
        if (!tile.valid) continue;
        const int m0 = tile.m_idx * BLOCK_M, n0 = tile.n_idx * BLOCK_N;
        int lo, hi;
        wgrad_range(p, group, lo, hi);
        if (p.accumulate && lo == hi) continue;
        if constexpr (SPLIT) {
            const int share = ceil_div(hi - lo, parts), end = hi;
            lo = min(lo + part * share, end);
            hi = min(lo + share, end);
        }
        // the ring is used again: everybody is out of it
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");

        // descriptors start at the tile and at the range's first column, so that 32-bit offsets reach whatever the operands' sizes
        const int rows_a = min(BLOCK_M, p.m - m0), rows_b = min(BLOCK_N, p.n - n0);
        const __amdgpu_buffer_rsrc_t rsrc_a = make_rsrc(p.a + size_t(m0) * p.k + size_t(lo) * 128, uint32_t(rows_a) * p.k - uint32_t(lo) * 128);
        const __amdgpu_buffer_rsrc_t rsrc_b = make_rsrc(p.b + size_t(n0) * p.k + size_t(lo) * 128, uint32_t(rows_b) * p.k - uint32_t(lo) * 128);
        // this wave's rows of scales: of a, of b, or (64 x 64) once more b's, which nobody reads; the last row stands for those behind it
        const bool of_a = wave < BLOCK_M / kWaveSize;
        const int ld_s = of_a ? p.ld_sa : p.ld_sb, rows_s = of_a ? rows_a : rows_b;
        const __amdgpu_buffer_rsrc_t rsrc_s = make_rsrc(of_a ? p.sa + size_t(m0) * ld_s : p.sb + size_t(n0) * ld_s, uint32_t(rows_s) * ld_s);
        const uint32_t off_s = uint32_t(min(wave * kWaveSize + lane - (of_a ? 0 : BLOCK_M), rows_s - 1)) * ld_s;
        StA stage_a;
        StB stage_b;
        stage_a.init(p.k, wave, lane);
        stage_b.init(p.k, wave, lane);
        stage_a.aim(rows_a, p.k, wave);
        stage_b.aim(rows_b, p.k, wave);
        const int count = hi - lo;
        // (behind the range's last k-tile there is none: the ring is used again below)
        auto copy = [&](int kt, int st) {
            if (kt >= count) return;
            uint8_t* const stage = ring + st * STAGE_BYTES;
            stage_a.issue(rsrc_a, stage, kt * kRowBytes, wave);
            stage_b.issue(rsrc_b, stage + A_BYTES, kt * kRowBytes, wave);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_s, YAN_LDS_PTR(ring_scales + st * SCALE_ROWS + wave * kWaveSize), 4, off_s, (lo + kt) & ~3, 0, 0);
        };
        // a lane reads chunks 2 g and 2 g + 1 of its row, sixteen codes each for two 16x16x32 MFMAs
        const int off[2] = {frag_offset<16>(lane, 2 * g), frag_offset<16>(lane, 2 * g + 1)};

        f32x4 acc[TN][TM];
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        // What a wave reads of a k-tile: sixteen codes a row and chunk, and the dwords with the rows' scales.
        struct Fragments {
            i32x4 a[2][TM], b[2][TN];
            uint32_t scales_a[TM], scales_b[TN];
        };
        auto read = [&](Fragments& f, int st) __attribute__((always_inline)) {
            const uint8_t* const pa = ring + st * STAGE_BYTES + wm * WTM * kRowBytes;
            const uint8_t* const pb = ring + st * STAGE_BYTES + A_BYTES + wn * WTN * kRowBytes;
            const uint32_t* const scales = ring_scales + st * SCALE_ROWS + col;
#pragma unroll
            for (int j = 0; j < TM; ++j) f.scales_a[j] = scales[wm * WTM + j * 16];
#pragma unroll
            for (int i = 0; i < TN; ++i) f.scales_b[i] = scales[BLOCK_M + wn * WTN + i * 16];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int j = 0; j < TM; ++j) f.a[c][j] = *reinterpret_cast<const i32x4*>(pa + j * 16 * kRowBytes + off[c]);
#pragma unroll
                for (int i = 0; i < TN; ++i) f.b[c][i] = *reinterpret_cast<const i32x4*>(pb + i * 16 * kRowBytes + off[c]);
            }
        };
        auto multiply = [&](const Fragments& f, int kt) __attribute__((always_inline)) {
            const int shift = (lo + kt) % 4 * 8;
            float scale_a[TM], scale_b[TN];
#pragma unroll
            for (int j = 0; j < TM; ++j) scale_a[j] = wgrad_scale(int(f.scales_a[j]), shift);
#pragma unroll
            for (int i = 0; i < TN; ++i) scale_b[i] = wgrad_scale(int(f.scales_b[i]), shift);
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    bf16x8 fa[TM], fb[TN];
#pragma unroll
                    for (int j = 0; j < TM; ++j) fa[j] = wgrad_decode(f.a[c][j][2 * h], f.a[c][j][2 * h + 1], scale_a[j]);
#pragma unroll
                    for (int i = 0; i < TN; ++i) fb[i] = wgrad_decode(f.b[c][i][2 * h], f.b[c][i][2 * h + 1], scale_b[i]);
#pragma unroll
                    for (int i = 0; i < TN; ++i)
#pragma unroll
                        for (int j = 0; j < TM; ++j) acc[i][j] = MfmaBF16_16x16x32::mma(fb[i], fa[j], acc[i][j]);
                }
        };
        // `ahead` stages behind the wanted one have been asked for, if the range has them
        auto landed = [&](auto ahead_c, bool all_there) __attribute__((always_inline)) {
            constexpr int AHEAD = decltype(ahead_c)::value;
            if (AHEAD > 0 && all_there) __builtin_amdgcn_s_waitcnt(waitcnt_imm(AHEAD * NUM_COPIES, 0));
            else __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        int st = 0;
        const auto behind = [](int at) { return at + 1 == STAGES ? 0 : at + 1; };
        if constexpr (BLOCK_M == 64) {
            // Fragments of the next k-tile are read while this one's are multiplied, so that a stage is free again as soon as it is begun (27 tiles of 199
            // k-tiles: 106 us, 95 so). Of the 0.48 us that a k-tile takes a workgroup alone on its compute unit 0.11 are MFMAs; 0.4 were left without conversions
            // and copies, for a barrier, the LDS, and chains of four MFMAs. Eight stages instead of four: no difference. The larger tile has no registers for it.
            Fragments f[2];
            for (int t = 0; t < STAGES; ++t) copy(t, t);
            if (count > 0) {
                landed(std::integral_constant<int, STAGES - 1>{}, count >= STAGES);
                read(f[0], 0);
            }
            auto step = [&](int kt, const Fragments& now, Fragments& next) __attribute__((always_inline)) {
                landed(std::integral_constant<int, STAGES - 2>{}, kt + STAGES <= count);
                copy(kt + STAGES, st);
                st = behind(st);
                if (kt + 1 < count) read(next, st);
                __builtin_amdgcn_sched_barrier(0);
                multiply(now, kt);
            };
            for (int kt = 0; kt < count; kt += 2) {
                step(kt, f[0], f[1]);
                if (kt + 1 < count) step(kt + 1, f[1], f[0]);
            }
        } else {
            for (int t = 0; t < STAGES - 1; ++t) copy(t, t);
            for (int kt = 0; kt < count; ++kt) {
                landed(std::integral_constant<int, STAGES - 2>{}, kt + STAGES - 2 < count);
                copy(kt + STAGES - 1, st == 0 ? STAGES - 1 : st - 1);
                Fragments f;
                read(f, st);
                multiply(f, kt);
                st = behind(st);
            }
        }

        // The 4 registers of atom (i, j) are columns 16 i + 4 g + {0..3} of row 16 j + col of the slab. Stored from there an instruction covers 16 rows by 64
        // bytes, half lines, which the memory takes at 3.2 to 4.8 TB/s; a wave turns its slab round through LDS and stores whole lines. Chunk c (16
        // bytes) of a row sits in slot c ^ row, so that neither side meets a bank twice.
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoWaitVm, 0));          // every wave has read the last k-tile
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (SPLIT && !wgrad_meet<NW>(acc, w, tile_slot, part, parts, wave, lane)) continue;
        constexpr int LANES_PER_ROW = WTN / 4, ROWS_PER_STORE = kWaveSize / LANES_PER_ROW, STORES = WTM / ROWS_PER_STORE;
        static_assert(NW * WTM * WTN * 4 <= STAGES * STAGE_BYTES && kWaveSize % LANES_PER_ROW == 0);
        uint8_t* const region = ring + wave * (WTM * WTN * 4);
        const auto place = [](int row, int chunk) { return row * (WTN * 4) + ((chunk ^ (row & (LANES_PER_ROW - 1))) * 16); };
        const int row_in = lane / LANES_PER_ROW, chunk = lane % LANES_PER_ROW;
        const bool stream_out = size_t(p.groups) * p.m * p.n * 4 > (size_t(32) << 20);
        const uint32_t row_bytes = uint32_t(p.n) * 4;
        const __amdgpu_buffer_rsrc_t rsrc_out = make_rsrc(p.out + (size_t(group) * p.m + m0) * p.n + n0, uint32_t(rows_a) * row_bytes - uint32_t(n0) * 4);
        const int c0 = wn * WTN + 4 * chunk;
        const uint32_t to = n0 + c0 < p.n ? uint32_t(wm * WTM + row_in) * row_bytes + uint32_t(c0) * 4 : kOutOfRange;
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
            wgrad_store(v, rsrc_out, to + u * ROWS_PER_STORE * row_bytes, stream_out);
        }
    }
}

// The large tiles: 256 x BLOCK_N on 4 waves, one per SIMD, each with a 128 x BLOCK_N / 2 slab of 16x16x32 MFMAs, its sums in the accumulation registers.
// A k-tile of 128 is four steps of 32; a step is TN rows of 8 MFMAs. A lone wave has nobody to hide behind, so everything else it issues stands in
// the shadow of an MFMA:
//   * a lane reads 16 codes of a row at a time, which are two steps: activation fragments are decoded one step ahead of their MFMAs (`mf`, two
//     buffers), weight fragments one row ahead (`nf`), one or two conversions behind every MFMA. The registers of the codes are read again as soon
//     as their second half is decoded, 7 rows or more before the next use;
//   * LDS holds two k-tiles. In the middle of k-tile t every wave has read all of t, and t + 1 has to have landed: one barrier a k-tile, in whose wake
//     the copies of t + 2 go out into the half that t leaves, one a row, with two steps to land after the last of them;
//   * scale bytes come as dwords of four k-tiles, loaded while the last k-tile that needs the old ones is under way, and become floats in the last
//     step of a k-tile, each where the next one's first fragment needs it;
//   * the walk is persistent (one workgroup per compute unit), and the stream of k-tiles does not stop at the end of a tile: the copies, scales and
//     first fragments of the next tile are under way when the sums of this one are stored.
// 64-bit bases per tile, 32-bit offsets inside.
struct WgradTile {
    int slot, group, m0, n0, lo, count;
};

template <int BLOCK_N>
__global__ void __launch_bounds__(256, 1)
fp8_wgrad_tall_kernel(WgradProblem p) {
    constexpr int BLOCK_M = 256, NW = 4, TM = 8, TN = BLOCK_N / 32, WTM = 128, WTN = BLOCK_N / 2;
    static_assert(BLOCK_N % 128 == 0 && TN >= 4 && TN <= 8);
    using StA = WgradStager<BLOCK_M, NW>;
    using StB = WgradStager<BLOCK_N, NW>;
    constexpr int A_BYTES = BLOCK_M * kRowBytes, STAGE_BYTES = (BLOCK_M + BLOCK_N) * kRowBytes, PASSES = StA::PASSES + StB::PASSES;
    static_assert(PASSES <= 3 * TN);            // a row of the step behind the barrier has two copies at most, of the one after it one
    // the sums leave through pieces of 16 rows by PIECE columns, two a wave
    constexpr int PIECE = 64, PIECE_BYTES = 16 * PIECE * 4, PIECES_PER_ROW = WTN / PIECE, PIECES = TM * PIECES_PER_ROW;
    constexpr int LANES_PER_ROW = PIECE / 4, ROWS_PER_STORE = kWaveSize / LANES_PER_ROW, PIECE_STORES = 16 / ROWS_PER_STORE;
    static_assert(WTN % PIECE == 0 && 2 * STAGE_BYTES + NW * 2 * PIECE_BYTES <= 160 * 1024);
    __shared__ __attribute__((aligned(1024))) uint8_t stages[2 * STAGE_BYTES + NW * 2 * PIECE_BYTES];
    uint8_t* const turn = stages + 2 * STAGE_BYTES;

    const XcdTileScheduler<> sched(p.m, p.n, BLOCK_M, BLOCK_N);
    const int per_group = sched.grid_size(), slots = per_group * p.groups;
    const int lane = get_lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int wn = wave % 2, wm = wave / 2, g = lane / 16, col = lane % 16;

    auto tile_at = [&](int slot) {
        WgradTile t{slot, 0, 0, 0, 0, 0};
        t.group = slot / per_group;
        const TileCoord c = sched.tile_of(slot - t.group * per_group);
        if (!c.valid) { t.count = -1; return t; }
        t.m0 = c.m_idx * BLOCK_M, t.n0 = c.n_idx * BLOCK_N;
        int hi;
        wgrad_range(p, t.group, t.lo, hi);
        t.count = hi - t.lo;
        return t;
    };
    // the next slot of this workgroup's walk, from `slot` on, whose tile has something to add up; count 0: the walk ends
    auto seek = [&](int slot) {
        for (; slot < slots; slot += gridDim.x) {
            const WgradTile t = tile_at(slot);
            if (t.count > 0) return t;
        }
        return WgradTile{slots, 0, 0, 0, 0, 0};
    };
    // the tiles of groups without columns
    if (p.offsets && !p.accumulate)
        for (int slot = blockIdx.x; slot < slots; slot += gridDim.x) {
            const WgradTile t = tile_at(slot);
            if (t.count != 0) continue;
            for (int r = wave; r < min(BLOCK_M, p.m - t.m0); r += NW) {
                float* const line = p.out + (size_t(t.group) * p.m + t.m0 + r) * p.n + t.n0;
                for (int c = 4 * lane; c < min(BLOCK_N, p.n - t.n0); c += 4 * kWaveSize) *reinterpret_cast<f32x4*>(line + c) = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }

    StA stage_a;
    StB stage_b;
    stage_a.init(p.k, wave, lane);
    stage_b.init(p.k, wave, lane);
    const int koff[2] = {frag_offset<16>(lane, 2 * g), frag_offset<16>(lane, 2 * g + 1)};
    const int a_lane = wm * WTM * kRowBytes, b_lane = A_BYTES + wn * WTN * kRowBytes;

    // What the copies read: k-tile `copy_kt` of `copy_tile`
    WgradTile copy_tile = seek(blockIdx.x);
    if (copy_tile.count == 0) return;
    WgradTile cur = copy_tile;
    int copy_kt = 0;
    __amdgpu_buffer_rsrc_t rsrc_a, rsrc_b;
    auto aim_copies = [&] {
        const WgradTile& t = copy_tile;
        const int rows_a = min(BLOCK_M, p.m - t.m0), rows_b = min(BLOCK_N, p.n - t.n0);
        rsrc_a = make_rsrc(p.a + size_t(t.m0) * p.k + size_t(t.lo) * 128, uint32_t(rows_a) * p.k - uint32_t(t.lo) * 128);
        rsrc_b = make_rsrc(p.b + size_t(t.n0) * p.k + size_t(t.lo) * 128, uint32_t(rows_b) * p.k - uint32_t(t.lo) * 128);
        stage_a.aim(rows_a, p.k, wave);
        stage_b.aim(rows_b, p.k, wave);
    };
    // Behind the walk's last k-tile that one is copied again, two times, into stages whose codes are not used any more: the count of copies under way stays
    // what the waits below take it for, and none is out of range.
    bool walking = true;
    auto advance_copies = [&] {
        if (!walking) return;
        if (++copy_kt < copy_tile.count) return;
        const WgradTile next = seek(copy_tile.slot + gridDim.x);
        walking = next.count != 0;
        if (!walking) {
            --copy_kt;
            return;
        }
        copy_tile = next, copy_kt = 0;
        aim_copies();
    };
    auto copy = [&](int d, int stage) __attribute__((always_inline)) {
        if (d < StA::PASSES) stage_a.issue_pass(rsrc_a, stages + stage, copy_kt * kRowBytes, wave, d);
        else stage_b.issue_pass(rsrc_b, stages + stage + A_BYTES, copy_kt * kRowBytes, wave, d - StA::PASSES);
    };
    // the dwords with the scales of k-tile `at` (counted from the start of K) of tile `t`
    int quad_a[TM], quad_b[TN];
    float sa[TM], sb[TN];
    auto load_scales = [&](const WgradTile& t, int at) __attribute__((always_inline)) {
        const int rows_a = t.count ? min(BLOCK_M, p.m - t.m0) : 0, rows_b = t.count ? min(BLOCK_N, p.n - t.n0) : 0;
        const __amdgpu_buffer_rsrc_t rsrc_sa = make_rsrc(p.sa + size_t(t.m0) * p.ld_sa, uint32_t(rows_a) * p.ld_sa);
        const __amdgpu_buffer_rsrc_t rsrc_sb = make_rsrc(p.sb + size_t(t.n0) * p.ld_sb, uint32_t(rows_b) * p.ld_sb);
#pragma unroll
        for (int j = 0; j < TM; ++j) quad_a[j] = __builtin_amdgcn_raw_buffer_load_b32(rsrc_sa, uint32_t(wm * WTM + col) * p.ld_sa, (at & ~3) + j * 16 * p.ld_sa, 0);
#pragma unroll
        for (int i = 0; i < TN; ++i) quad_b[i] = __builtin_amdgcn_raw_buffer_load_b32(rsrc_sb, uint32_t(wn * WTN + col) * p.ld_sb, (at & ~3) + i * 16 * p.ld_sb, 0);
    };

    f32x4 acc[TN][TM];
    i32x4 raw_m[TM], raw_n[TN], mf[2][TM], nf[2];
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    // two codes; the empty asm keeps the conversion where it stands (the compiler would move it down to its use, in front of the MFMA)
    auto decode = [](int codes, float scale, bool upper) __attribute__((always_inline)) {
        int two = __builtin_bit_cast(int, upper ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(codes), scale, true)
                                                : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(codes), scale, false));
        asm volatile("" : "+v"(two));
        return two;
    };
    auto mma = [&](auto first_c, int q, int i, int j) __attribute__((always_inline)) {
        f32x4& sum = acc[i][j];
        const i32x4 &n = nf[i & 1], &m = mf[q & 1][j];
        if constexpr (decltype(first_c)::value) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=a"(sum) : "v"(n), "v"(m));
        else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(sum) : "v"(n), "v"(m));
    };
    auto read_m = [&](int j, int stage, int set) __attribute__((always_inline)) {
        raw_m[j] = *reinterpret_cast<const i32x4*>(stages + stage + a_lane + j * 16 * kRowBytes + koff[set]);
    };
    auto read_n = [&](int i, int stage, int set) __attribute__((always_inline)) {
        raw_n[i] = *reinterpret_cast<const i32x4*>(stages + stage + b_lane + i * 16 * kRowBytes + koff[set]);
    };
    auto float_scale = [](int quad, int shift) __attribute__((always_inline)) {
        float scale = wgrad_scale(quad, shift);
        asm volatile("" : "+v"(scale));
        return scale;
    };

    // Step Q of the k-tile staged at `here`; the next one is staged at `there`, its scales are in the dwords at bit `shift`. FIRST: the sums start here.
    auto step = [&](auto first_c, auto q_c, int here, int there, int shift) __attribute__((always_inline)) {
        constexpr int Q = decltype(q_c)::value;
        constexpr bool EVEN = Q % 2 == 0;
        // the codes read in steps 0 and 1 are the second set of this k-tile, in steps 2 and 3 the first set of the next
        const int from = Q < 2 ? here : there;
        constexpr int SET = Q < 2 ? 1 : 0;
        // the next step's fragments lie in the half of their 16 codes that its number says
        constexpr int M_HALF = (Q + 1) % 2;
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const int next = i + 1 < TN ? i + 1 : 0, n_half = i + 1 < TN ? Q % 2 : M_HALF;      // weight row decoded behind this one's MFMAs
            const bool more = i + TN < TM;                                                      // fewer rows than activation fragments: two in one row
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                mma(first_c, Q, i, j);
                if (j < 4) {
                    nf[next & 1][j] = decode(raw_n[next][2 * n_half + j / 2], sb[next], j % 2);
                    if (more) mf[M_HALF][(i + TN) % TM][j] = decode(raw_m[(i + TN) % TM][2 * M_HALF + j / 2], sa[(i + TN) % TM], j % 2);
                } else {
                    mf[M_HALF][i][j - 4] = decode(raw_m[i][2 * M_HALF + (j - 4) / 2], sa[i], j % 2);
                }
                if (EVEN && j == 1 && i > 0) {          // both halves of these are decoded
                    read_m(i - 1, from, SET);
                    if (i - 1 + TN < TM) read_m((i - 1 + TN) % TM, from, SET);
                }
                if (!EVEN && j == 2 && i == 0) {
                    read_m(TN - 1, from, SET);
                    if (2 * TN - 1 < TM) read_m((2 * TN - 1) % TM, from, SET);
                }
                if (!EVEN && j == 1) read_n(i, from, SET);
                if (Q >= 2 && j == 5 && (Q - 2) * TN + i < PASSES) copy((Q - 2) * TN + i, here);
                if (Q == 2 && j == 3 && 2 * TN + i < PASSES) copy(2 * TN + i, here);
                if (Q == 2 && j == 6 && more) sa[(i + TN) % TM] = float_scale(quad_a[(i + TN) % TM], shift);
                if (Q == 3 && j == 3) sa[i] = float_scale(quad_a[i], shift);
                if (Q == 3 && j == 6) sb[i] = float_scale(quad_b[i], shift);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    using Q0 = std::integral_constant<int, 0>;
    using Q1 = std::integral_constant<int, 1>;
    using Q2 = std::integral_constant<int, 2>;
    using Q3 = std::integral_constant<int, 3>;
    constexpr int STORES = PIECES * PIECE_STORES;       // of a tile, by every wave, whatever of it exists

    // the first two k-tiles of the walk, the scales and first fragments of the first
    aim_copies();
    for (int s = 0; s < 2; ++s) {
        for (int d = 0; d < StA::PASSES; ++d) copy(d, s * STAGE_BYTES);
        for (int d = 0; d < StB::PASSES; ++d) copy(StA::PASSES + d, s * STAGE_BYTES);
        advance_copies();
    }
    load_scales(cur, cur.lo);
    {
        const int shift = cur.lo % 4 * 8;
#pragma unroll
        for (int j = 0; j < TM; ++j) sa[j] = float_scale(quad_a[j], shift);
#pragma unroll
        for (int i = 0; i < TN; ++i) sb[i] = float_scale(quad_b[i], shift);
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < TM; ++j) read_m(j, 0, 0);
#pragma unroll
    for (int i = 0; i < TN; ++i) read_n(i, 0, 0);
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) mf[0][j][w] = decode(raw_m[j][w / 2], sa[j], w % 2);
#pragma unroll
    for (int w = 0; w < 4; ++w) nf[0][w] = decode(raw_n[0][w / 2], sb[0], w % 2);
    __builtin_amdgcn_sched_barrier(0);

    const bool stream_out = size_t(p.groups) * p.m * p.n * 4 > (size_t(32) << 20);
    const uint32_t row_bytes = uint32_t(p.n) * 4;
    int here = 0;
    while (true) {
        const WgradTile nxt = seek(cur.slot + gridDim.x);
        auto k_tile = [&](auto first_c, int kt) __attribute__((always_inline)) {
            const bool last = kt + 1 == cur.count;
            const int next_at = last ? nxt.lo : cur.lo + kt + 1, shift = next_at % 4 * 8, there = STAGE_BYTES - here;
            if (last) load_scales(nxt, next_at);
            else if (next_at % 4 == 0) load_scales(cur, next_at);
            step(first_c, Q0{}, here, there, shift);
            step(std::false_type{}, Q1{}, here, there, shift);
            // k-tile t + 1 has landed, and every wave has read k-tile t. Behind the copies of t + 1 a wave has issued nothing, or, in a tile's
            // first k-tile, the stores of the tile before, which need not be done.
            __builtin_amdgcn_s_waitcnt(waitcnt_imm(decltype(first_c)::value ? (STORES < 63 ? STORES : 63) : 0, 0));
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            step(std::false_type{}, Q2{}, here, there, shift);
            step(std::false_type{}, Q3{}, here, there, shift);
            advance_copies();
            here = there;
        };
        k_tile(std::true_type{}, 0);
        for (int kt = 1; kt < cur.count; ++kt) k_tile(std::false_type{}, kt);
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");      // the last MFMAs retire before the sums are read

        // The 4 registers of atom (i, j) are columns 16 i + 4 g + {0..3} of row 16 j + col of the slab. A wave turns it round through LDS of its own, 16
        // rows by PIECE columns at a time and two such pieces in turn: the sums of piece u go in, piece u - 1 comes out as runs of whole lines,
        // piece u - 2 is stored. Chunk c (16 bytes) of a row sits in slot c ^ row. Every wave issues all STORES stores, those outside of the output out
        // of range.
        auto epilogue = [&](auto policy_c, auto accumulate_c) __attribute__((always_inline)) {
            constexpr bool ACCUMULATE = decltype(accumulate_c)::value;
            constexpr int AHEAD = 2;            // pieces of what is added to that are under way
            uint8_t* const buffers = turn + wave * (2 * PIECE_BYTES);
            const __amdgpu_buffer_rsrc_t rsrc_out = make_rsrc(p.out + (size_t(cur.group) * p.m + cur.m0) * p.n + cur.n0,
                                                              uint32_t(min(BLOCK_M, p.m - cur.m0)) * row_bytes - uint32_t(cur.n0) * 4);
            const int row_in = lane / LANES_PER_ROW, chunk = lane % LANES_PER_ROW;
            uint32_t off[PIECES_PER_ROW];
#pragma unroll
            for (int h = 0; h < PIECES_PER_ROW; ++h) {
                const int c = wn * WTN + PIECE * h + 4 * chunk;
                off[h] = cur.n0 + c < p.n ? uint32_t(wm * WTM + row_in) * row_bytes + uint32_t(c) * 4 : kOutOfRange;
            }
            i32x4 back[2][PIECE_STORES], held[ACCUMULATE ? AHEAD + 1 : 1][PIECE_STORES];
            auto load = [&](int u) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < PIECE_STORES; ++s)
                    held[u % (AHEAD + 1)][s] = __builtin_amdgcn_raw_buffer_load_b128(rsrc_out, off[u % PIECES_PER_ROW], (u / PIECES_PER_ROW * 16 + ROWS_PER_STORE * s) * row_bytes, 0);
            };
            if constexpr (ACCUMULATE) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) load(u);
            }
#pragma unroll
            for (int u = 0; u < PIECES + 2; ++u) {
                if (u < PIECES) {
                    const int j = u / PIECES_PER_ROW, h = u % PIECES_PER_ROW;
#pragma unroll
                    for (int a = 0; a < PIECE / 16; ++a) {
                        const f32x4& sum = acc[h * (PIECE / 16) + a][j];
                        f32x4 v;
                        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[0]) : "a"(sum[0]));
                        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[1]) : "a"(sum[1]));
                        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[2]) : "a"(sum[2]));
                        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[3]) : "a"(sum[3]));
                        *reinterpret_cast<f32x4*>(buffers + (u & 1) * PIECE_BYTES + col * (PIECE * 4) + (((4 * a + g) ^ (col & (LANES_PER_ROW - 1))) * 16)) = v;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                if (u >= 1 && u - 1 < PIECES) {
#pragma unroll
                    for (int s = 0; s < PIECE_STORES; ++s) {
                        const int row = ROWS_PER_STORE * s + row_in;
                        back[(u - 1) & 1][s] = *reinterpret_cast<const i32x4*>(buffers + ((u - 1) & 1) * PIECE_BYTES + row * (PIECE * 4) + ((chunk ^ (row & (LANES_PER_ROW - 1))) * 16));
                    }
                }
                if (u >= 2) {
                    const int w = u - 2;
                    if constexpr (ACCUMULATE) {
                        if (w + AHEAD < PIECES) load(w + AHEAD);
                    }
#pragma unroll
                    for (int s = 0; s < PIECE_STORES; ++s) {
                        f32x4 v = __builtin_bit_cast(f32x4, back[w & 1][s]);
                        if constexpr (ACCUMULATE) v += __builtin_bit_cast(f32x4, held[w % (AHEAD + 1)][s]);
                        wgrad_store(v, rsrc_out, off[w % PIECES_PER_ROW] + (w / PIECES_PER_ROW * 16 + ROWS_PER_STORE * s) * row_bytes, decltype(policy_c)::value);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        using Kept = std::false_type;
        using Streamed = std::true_type;
        if (p.accumulate) {
            if (stream_out) epilogue(Streamed{}, std::true_type{});
            else epilogue(Kept{}, std::true_type{});
        } else {
            if (stream_out) epilogue(Streamed{}, std::false_type{});
            else epilogue(Kept{}, std::false_type{});
        }
        if (nxt.count == 0) break;
        cur = nxt;
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(STORES < 63 ? STORES : 63, 0));         // the copies behind the last k-tile have landed: the LDS may be another's from here on
}

// Which kernel a problem runs on, and in how many parts its K ranges. Every kernel was timed on 246 shapes (32 to 8192 rows and columns, 1 to 199 k-tiles, 1
// to 64 groups); the choice is 0.8 % slower than the fastest on average, 1.4 % over 163 others drawn afterwards.
//   * Up to two 64 x 64 tiles a compute unit run those, in 2 parts as long as that is two workgroups a compute unit (counted as launched, a multiple of 8 a
//     group), in 4, 8 or 16 as long as it is one, and from 12, 12, 24 and 64 k-tiles on (us whole, in 2, 4, 8: 64 tiles of 64 k-tiles 33, 21, 14.6, 15.8; 27
//     of 199 95, 52, 29.5, 19.8).
//   * Others by an estimate in us. 256 x 256: rounds over the chip times 2.6 a k-tile and 12 for the output, 20 accumulated, which a lone workgroup stores with
//     little else to do, and 4 for the start. 256 x 128: 1.3, 8 and 12.5. 128 x 128 and 64 x 64, two workgroups on a compute unit: 1.65 and 0.66 a k-tile, 6 and
//     2.5 for the output; alone on one, as in a last round of one workgroup a compute unit or less, 1.1 and 0.47. (99 k-tiles of 2048 x 4096: 228, 157 and 186;
//     512 x 512, 5 k-tiles of 64 groups: 55, 38 and 35; 7168 tiles of 256 x 256 and 5 k-tiles 575 / 732 for 128 x 128, accumulated 1036 / 1044.) The large tiles have
//     to be 8 % ahead.
enum WgradKernel { kWgradAny, kWgradTall, kWgradMiddle, kWgrad128, kWgrad64, kWgradSplit };
struct WgradPlan {
    WgradKernel kernel;
    int parts;
};
constexpr long long kWgradMostParts = (kSplitKWorkspaceBytes - kSplitKCounterBytes) / (64 * 64 * 4);        // what a workspace holds, sums and counters
static_assert(kWgradMostParts * 4 * 4 <= (long long)kSplitKCounterBytes);
inline WgradPlan wgrad_plan(int m, int n, int k, int groups, bool accumulate, int num_cus, bool may_split) {
    const auto tiles = [&](int block_m, int block_n) { return (long long)ceil_div(m, block_m) * ceil_div(n, block_n) * groups; };
    const double k_tiles = double(k / 128) / groups;
    const long long small = tiles(64, 64);
    if (small <= 2ll * num_cus) {
        const long long slots = (long long)XcdTileScheduler<>(m, n, 64, 64).grid_size() * groups;
        const struct { int parts, per_cu; double k_tiles; } ways[] = {{16, 1, 64}, {8, 1, 24}, {4, 1, 12}, {2, 2, 12}};
        for (const auto& way : ways)
            if (may_split && slots * way.parts <= (long long)way.per_cu * num_cus && k_tiles >= way.k_tiles && slots * way.parts <= kWgradMostParts)
                return {kWgradSplit, way.parts};
        return {kWgrad64, 1};
    }
    const double rounds = double(ceil_div(tiles(256, 256), (long long)num_cus)), rounds_middle = double(ceil_div(tiles(256, 128), (long long)num_cus));
    const double tall = 4 + rounds * (2.6 * k_tiles + (accumulate ? 20 : 12)), middle = rounds_middle * (1.3 * k_tiles + (accumulate ? 12.5 : 8));
    const auto in_twos = [&](long long count, double two, double one) {
        const long long rest = count % (2 * num_cus);
        return double(count / (2 * num_cus)) * two + (rest == 0 ? 0. : rest <= num_cus ? one : two);
    };
    const double flat = in_twos(tiles(128, 128), 1.65 * k_tiles + (accumulate ? 9.5 : 6), 1.1 * k_tiles + (accumulate ? 4.5 : 3.5));
    const double least = 2 + in_twos(small, 0.66 * k_tiles + (accumulate ? 3.5 : 2.5), 0.47 * k_tiles + (accumulate ? 2 : 1.5));
    if (std::min(tall, middle) < 0.92 * std::min(flat, least)) return {tall < middle ? kWgradTall : kWgradMiddle, 1};
    return {flat < least ? kWgrad128 : kWgrad64, 1};
}

// m, n, k: codes a [m, k], b [n, k], n % 4 == 0, k % 128 == 0; scale rows ld_sa, ld_sb bytes apart (multiples of 4, k / 128 rounded up to 4 or more),
// 4-byte aligned; out [groups, m, n], 16-byte aligned. offsets null: groups is 1. `workspace`: a split-K workspace (kSplitKWorkspaceBytes, its
// counters zero), or null: K is not split. num_sms: compute units to use, 0 for all.
template <WgradKernel KERNEL = kWgradAny, int PARTS = 1>
inline hipError_t launch_fp8_wgrad(const void* a, const uint8_t* sa, int ld_sa, const void* b, const uint8_t* sb, int ld_sb, float* out, const int* offsets,
                                   int groups, int m, int n, int k, bool accumulate, void* workspace, int num_sms, hipStream_t stream) {
    if (m < 0 || n < 0 || n % 4 != 0 || k < 0 || k % 128 != 0 || groups < 0 || (!offsets && groups != 1)) return hipErrorInvalidValue;
    if (k >= 1 << 23 || n >= 1 << 21 || ld_sa % 4 != 0 || ld_sb % 4 != 0 || ld_sa >= 1 << 23 || ld_sb >= 1 << 23) return hipErrorInvalidValue;
    if (ld_sa < ceil_div(k / 128, 4) * 4 || ld_sb < ceil_div(k / 128, 4) * 4) return hipErrorInvalidValue;
    if (m == 0 || n == 0 || groups == 0) return hipSuccess;
    if (!out || (k && (!a || !b || !sa || !sb))) return hipErrorInvalidValue;
    const WgradProblem p{static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(b), sa, sb, out, offsets, m, n, k, ld_sa, ld_sb, groups, accumulate};
    const bool capped = num_sms > 0 && num_sms < device_cu_count();
    const int cus = capped ? num_sms : device_cu_count();
    const WgradPlan plan = KERNEL == kWgradAny ? wgrad_plan(m, n, k, groups, accumulate, cus, workspace != nullptr) : WgradPlan{KERNEL, PARTS};
    const int block_m = plan.kernel == kWgradTall || plan.kernel == kWgradMiddle ? 256 : plan.kernel == kWgrad128 ? 128 : 64;
    const int block_n = plan.kernel == kWgradMiddle ? 128 : block_m;
    const long long slots = (long long)XcdTileScheduler<>(m, n, block_m, block_n).grid_size() * groups * plan.parts;
    if (slots >= 1ll << 24) return hipErrorInvalidValue;          // a launch has less than 2^32 threads
    WgradWorkspace w{nullptr, nullptr};
    if (plan.kernel == kWgradSplit) {
        if (!workspace || slots > kWgradMostParts) return hipErrorInvalidValue;
        w = {reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kSplitKCounterBytes), static_cast<unsigned*>(workspace)};
    }
    const auto launch = [&](auto kernel, long long grid, auto... more) {
        hipLaunchKernelGGL(kernel, dim3(uint32_t(grid)), dim3(256), 0, stream, p, more...);
        return hipGetLastError();
    };
    const long long most = capped ? std::min<long long>(cus, slots) : slots;
    switch (plan.kernel) {
        case kWgradTall: return launch(fp8_wgrad_tall_kernel<256>, std::min<long long>(cus, slots));
        case kWgradMiddle: return launch(fp8_wgrad_tall_kernel<128>, std::min<long long>(cus, slots));
        case kWgrad128: return launch(fp8_wgrad_kernel<128, 128, 2, false>, most, w, 1);
        case kWgrad64: return launch(fp8_wgrad_kernel<64, 64, 4, false>, most, w, 1);
        default: return launch(fp8_wgrad_kernel<64, 64, 4, true>, most, w, plan.parts);
    }
}

} // namespace yan
