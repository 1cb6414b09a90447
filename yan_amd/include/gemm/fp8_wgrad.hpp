// out[i, j] (+)= sum_b 2^(sa[i, b] + sb[j, b] - 254) sum_{t < 128} a[i, 128 b + t] b[j, 128 b + t]      (e4m3 x e4m3 -> fp32)
//
// The product of a weight gradient: both operands quantised 1 x 128 along K, which is the tokens, with power-of-two scales, the sums
// in fp32 and added to what is in `out` if asked. Grouped: K is cut at `offsets` (multiples of 128, on the device) and group g has its own
// out[g], the gradient of one expert's weights.
//
// The codes are multiplied as bf16, which holds code * 2^e exactly: gfx950 converts two codes and applies a power of two in one instruction, so
// the scales cost nothing and the sums stay in the matrix core's accumulators from the first k-tile to the last. The FP8 MFMAs are twice as
// fast and add up less exactly than fp32 sums do: small products next to large ones lose bits inside of the instruction, whatever its shape
// and also from a zero accumulator, 1.3e-5 of the result's norm for normal operands and 6e-5 where values spread more widely (bf16: 1e-7).
// A gradient that is summed up in fp32 over micro-batches is to keep what fp32 keeps.
//
// Tiles are staged as in the other GEMMs (tile_io.hpp): 128-byte rows, swizzled, HBM -> LDS directly, in a ring. A row's scale bytes lie
// along K, rows a multiple of 4 bytes apart, so a lane loads those of four k-tiles as a dword.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_fp8.h>

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

// K range of a group in k-tiles. Offsets are the caller's, on the device: whatever they hold, the range lies inside K.
__device__ __forceinline__ void wgrad_range(const WgradProblem& p, int group, int& lo, int& hi) {
    const int k_tiles = p.k / 128;
    lo = 0, hi = k_tiles;
    if (p.offsets) {
        lo = min(max(p.offsets[group], 0) / 128, k_tiles);
        hi = max(lo, min(max(p.offsets[group + 1], 0) / 128, k_tiles));
    }
}

// Eight codes times a power of two (a float, of which the exponent counts) as bf16.
__device__ __forceinline__ bf16x8 wgrad_decode(int lo, int hi, float scale) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(lo), scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(lo), scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(hi), scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(hi), scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The scale of a k-tile out of the dword that holds those of four: `shift` is 8 times its place.
__device__ __forceinline__ float wgrad_scale(int quad, int shift) { return __builtin_bit_cast(float, ((uint32_t(quad) >> shift) & 0xff) << 23); }

template <int BLOCK_M, int BLOCK_N, int STAGES>
__global__ void __launch_bounds__(256)
fp8_wgrad_kernel(WgradProblem p) {
    constexpr int NW = 4, WTM = BLOCK_M / 2, WTN = BLOCK_N / 2, TM = WTM / 32, TN = WTN / 32;
    using StA = TileStager<BLOCK_M, NW>;
    using StB = TileStager<BLOCK_N, NW>;
    constexpr int NUM_COPIES = StA::PASSES + StB::PASSES, A_BYTES = BLOCK_M * kRowBytes, STAGE_BYTES = (BLOCK_M + BLOCK_N) * kRowBytes;
    static_assert(StA::PADDED_ROWS == BLOCK_M && StB::PADDED_ROWS == BLOCK_N && (STAGES - 2) * NUM_COPIES <= 63);
    __shared__ __attribute__((aligned(1024))) uint8_t ring[STAGES * STAGE_BYTES];

    const XcdTileScheduler<> sched(p.m, p.n, BLOCK_M, BLOCK_N);
    const int slots = sched.grid_size(), group = blockIdx.x / slots;
    const TileCoord tile = sched.tile_of(blockIdx.x % slots);
    if (!tile.valid) return;
    const int m0 = tile.m_idx * BLOCK_M, n0 = tile.n_idx * BLOCK_N;
    int lo, hi;
    wgrad_range(p, group, lo, hi);
    if (p.accumulate && lo == hi) return;

    const int lane = get_lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int wn = wave % 2, wm = wave / 2, g = lane / 32, row = lane % 32;
    // descriptors start at the tile and at the group's first column, so that 32-bit offsets reach whatever the operands' sizes
    const int rows_a = min(BLOCK_M, p.m - m0), rows_b = min(BLOCK_N, p.n - n0);
    const __amdgpu_buffer_rsrc_t rsrc_a = make_rsrc(p.a + size_t(m0) * p.k + size_t(lo) * 128, uint32_t(rows_a) * p.k - uint32_t(lo) * 128);
    const __amdgpu_buffer_rsrc_t rsrc_b = make_rsrc(p.b + size_t(n0) * p.k + size_t(lo) * 128, uint32_t(rows_b) * p.k - uint32_t(lo) * 128);
    const __amdgpu_buffer_rsrc_t rsrc_none = make_rsrc(p.a, 0);
    const __amdgpu_buffer_rsrc_t rsrc_sa = make_rsrc(p.sa + size_t(m0) * p.ld_sa, uint32_t(rows_a) * p.ld_sa);
    const __amdgpu_buffer_rsrc_t rsrc_sb = make_rsrc(p.sb + size_t(n0) * p.ld_sb, uint32_t(rows_b) * p.ld_sb);
    StA stage_a;
    StB stage_b;
    stage_a.init(0, p.k, wave, lane);
    stage_b.init(0, p.k, wave, lane);
    const int count = hi - lo;
    auto copy = [&](int kt, uint8_t* stage) {
        const bool live = kt < count;
        stage_a.issue(live ? rsrc_a : rsrc_none, stage, kt * kRowBytes, wave);
        stage_b.issue(live ? rsrc_b : rsrc_none, stage + A_BYTES, kt * kRowBytes, wave);
    };
    // a lane reads chunks 2 c + g of its row, c = 0 .. 3: eight codes each for two 32x32x16 MFMAs
    int off[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) off[c] = frag_offset<32>(lane, 2 * c + g);

    f32x16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    for (int t = 0; t < STAGES - 1; ++t) copy(t, ring + t * STAGE_BYTES);
    int st = 0, quad_a[TM], quad_b[TN];
    for (int kt = 0; kt < count; ++kt) {
        const int at = lo + kt;
        if (kt == 0 || at % 4 == 0) {
#pragma unroll
            for (int j = 0; j < TM; ++j) quad_a[j] = __builtin_amdgcn_raw_buffer_load_b32(rsrc_sa, uint32_t(wm * WTM + j * 32 + row) * p.ld_sa, at & ~3, 0);
#pragma unroll
            for (int i = 0; i < TN; ++i) quad_b[i] = __builtin_amdgcn_raw_buffer_load_b32(rsrc_sb, uint32_t(wn * WTN + i * 32 + row) * p.ld_sb, at & ~3, 0);
        }
        // every wave has as many copies under way: at most those of the STAGES - 2 k-tiles behind this one are left out here
        __builtin_amdgcn_s_waitcnt(waitcnt_imm((STAGES - 2) * NUM_COPIES, 0));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        copy(kt + STAGES - 1, ring + (st == 0 ? STAGES - 1 : st - 1) * STAGE_BYTES);
        const uint8_t* pa = ring + st * STAGE_BYTES + wm * WTM * kRowBytes;
        const uint8_t* pb = ring + st * STAGE_BYTES + A_BYTES + wn * WTN * kRowBytes;
        const int shift = at % 4 * 8;
        float scale_a[TM], scale_b[TN];
#pragma unroll
        for (int j = 0; j < TM; ++j) scale_a[j] = wgrad_scale(quad_a[j], shift);
#pragma unroll
        for (int i = 0; i < TN; ++i) scale_b[i] = wgrad_scale(quad_b[i], shift);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            i32x4 raw_a[TM], raw_b[TN];
#pragma unroll
            for (int j = 0; j < TM; ++j) raw_a[j] = *reinterpret_cast<const i32x4*>(pa + j * 32 * kRowBytes + off[c]);
#pragma unroll
            for (int i = 0; i < TN; ++i) raw_b[i] = *reinterpret_cast<const i32x4*>(pb + i * 32 * kRowBytes + off[c]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                bf16x8 fa[TM], fb[TN];
#pragma unroll
                for (int j = 0; j < TM; ++j) fa[j] = wgrad_decode(raw_a[j][2 * h], raw_a[j][2 * h + 1], scale_a[j]);
#pragma unroll
                for (int i = 0; i < TN; ++i) fb[i] = wgrad_decode(raw_b[i][2 * h], raw_b[i][2 * h + 1], scale_b[i]);
#pragma unroll
                for (int i = 0; i < TN; ++i)
#pragma unroll
                    for (int j = 0; j < TM; ++j) acc[i][j] = MfmaBF16_32x32x16::mma(fb[i], fa[j], acc[i][j]);
            }
        }
        st = st + 1 == STAGES ? 0 : st + 1;
    }

    // registers 4 q .. 4 q + 3 of atom (i, j): columns 8 q + 4 g + {0..3} of row `row`
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int mm = m0 + wm * WTM + j * 32 + row;
        if (mm >= p.m) continue;
        float* const line = p.out + (size_t(group) * p.m + mm) * p.n;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int nn = n0 + wn * WTN + i * 32 + 8 * q + 4 * g;
                if (nn >= p.n) continue;
                f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                f32x4* const to = reinterpret_cast<f32x4*>(line + nn);
                if (p.accumulate) v += *to;
                *to = v;
            }
    }
}

// m, n, k: codes a [m, k], b [n, k], n % 4 == 0, k % 128 == 0; scale rows ld_sa, ld_sb bytes apart (multiples of 4, k / 128 rounded up to 4 or more),
// 4-byte aligned; out [groups, m, n], 16-byte aligned. offsets null: groups is 1.
template <int = 0>
inline hipError_t launch_fp8_wgrad(const void* a, const uint8_t* sa, int ld_sa, const void* b, const uint8_t* sb, int ld_sb, float* out, const int* offsets,
                                   int groups, int m, int n, int k, bool accumulate, hipStream_t stream) {
    if (m < 0 || n < 0 || n % 4 != 0 || k < 0 || k % 128 != 0 || groups < 0 || (!offsets && groups != 1)) return hipErrorInvalidValue;
    if (k >= 1 << 23 || ld_sa % 4 != 0 || ld_sb % 4 != 0 || ld_sa < ceil_div(k / 128, 4) * 4 || ld_sb < ceil_div(k / 128, 4) * 4 || ld_sa >= 1 << 23 || ld_sb >= 1 << 23) return hipErrorInvalidValue;
    if (m == 0 || n == 0 || groups == 0) return hipSuccess;
    if (!out || (k && (!a || !b || !sa || !sb))) return hipErrorInvalidValue;
    const WgradProblem p{static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(b), sa, sb, out, offsets, m, n, k, ld_sa, ld_sb, groups, accumulate};
    const long long slots = XcdTileScheduler<>(m, n, 128, 128).grid_size();
    if (slots * groups >= 1ll << 31) return hipErrorInvalidValue;
    hipLaunchKernelGGL((fp8_wgrad_kernel<128, 128, 4>), dim3(uint32_t(slots * groups)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

} // namespace yan
