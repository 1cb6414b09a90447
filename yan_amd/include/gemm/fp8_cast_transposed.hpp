// The quantiser in front of a weight gradient: x [m, n] -> e4m3 codes [n, m'], one power-of-two scale for every 128 of a column's rows.
//
//   column j, rows 128 b .. 128 b + 127:  amax = max |x|, at least 2^-100;  e = the smallest with amax <= 448 * 2^e;
//   code = e4m3(x * 2^-e), round to nearest even;  the scale is kept as the byte e + 127 (E8M0), the form the scaled MFMAs take
//
// A weight gradient contracts over tokens, so both of its operands need their tokens contiguous: the kernel turns them round on the way. With
// `source`, row r of the result is x[source[r]] or, where that is none of x's rows, zeros: activations go from the tokens' order straight to the
// experts' rows. Without, rows from m on are zeros. x * 2^-e is exact, so the code is the nearest to x there is at this scale. NaN and
// infinity become NaN codes and do not count for amax.
//
// Bound by HBM: (2 or 4) bytes read and one written per element. A workgroup takes 128 rows (one scale) of 64 columns, a line of
// bf16 a row; a thread has four neighbouring rows of eight columns, whose codes are a dword each in LDS, column by column, from
// where they leave as whole lines.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include "fp8_cast.hpp"

namespace yan {

constexpr int kCastColumns = 64;
constexpr long long kCastPastBytes = 64ll << 20;

// Four rows of eight columns of a thread, and what is done with them; `columns` by their place among the thread's eight.
//   sizes        the columns' largest magnitudes, as bits, without what is not finite
//   exponents    e + 127 of the smallest e with amax <= 448 * 2^e: 448 = 1.75 * 2^8, so that what adding 0x1f.. to the bits carries into the exponent is
//                the one more that a mantissa above 1.75 asks for
//   four codes   of a column's rows, by the conversion that divides by a power of two itself (the exponent of its operand)
template <int BYTES> struct CastTile;         // of an element: 2, bf16, or 4, fp32

template <> struct CastTile<2> {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    i32x4 w[4];                         // dword d: columns 2 d and 2 d + 1
    i32x4 size;
    __device__ __forceinline__ static int column(int part, int c) { return 8 * part + c; }
    __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
    }
    __device__ __forceinline__ void sizes() {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t a = uint32_t(w[0][d]) & 0x7fff7fffu;
#pragma unroll
            for (int r = 1; r < 4; ++r) a = larger(a, uint32_t(w[r][d]) & 0x7fff7fffu);
            size[d] = int(a);
        }
        const uint32_t all = larger(larger(uint32_t(size[0]), uint32_t(size[1])), larger(uint32_t(size[2]), uint32_t(size[3])));
        if (__any((all & 0xffff) >= 0x7f80 || (all >> 16) >= 0x7f80)) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                uint32_t a = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t bits = uint32_t(w[r][d]) & 0x7fff7fffu;
                    a = larger(a, ((bits & 0xffff) >= 0x7f80 ? 0 : bits & 0xffff) | ((bits >> 16) >= 0x7f80 ? 0 : bits & 0xffff0000u));
                }
                size[d] = int(a);
            }
        }
    }
    static constexpr int SIZES = 4;
    __device__ __forceinline__ uint32_t& size_at(int i) { return reinterpret_cast<uint32_t*>(&size)[i]; }
    // of the 64 columns' sizes as the waves leave them, column `j`'s; and the exponent for it
    __device__ __forceinline__ static uint32_t size_in(const uint32_t* sizes, int j) { return reinterpret_cast<const uint16_t*>(sizes)[j]; }
    __device__ __forceinline__ static int exponent_of(uint32_t size) { return int((larger(size, 0x0d80u) + 0x1fu) >> 7) - 8; }
    __device__ __forceinline__ int exponent(int c) const {
        const uint32_t least = 0x0d800d80u;             // 2^-100
        const u16x2 e = ((__builtin_bit_cast(u16x2, larger(uint32_t(size[c / 2]), least)) + uint16_t(0x1f)) >> uint16_t(7)) - uint16_t(8);
        return e[c % 2];
    }
    __device__ __forceinline__ int codes(int c, int e) const {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        typedef short i16x2 __attribute__((ext_vector_type(2)));
        const uint32_t pick = c % 2 ? 0x07060302u : 0x05040100u;
        const float scale = __builtin_bit_cast(float, e << 23);
        i16x2 q{0, 0};
        q = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(q, __builtin_bit_cast(bf16x2, __builtin_amdgcn_perm(uint32_t(w[1][c / 2]), uint32_t(w[0][c / 2]), pick)), scale, false);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(q, __builtin_bit_cast(bf16x2, __builtin_amdgcn_perm(uint32_t(w[3][c / 2]), uint32_t(w[2][c / 2]), pick)), scale, true);
        return __builtin_bit_cast(int, q);
    }
};

template <> struct CastTile<4> {
    i32x4 w[8];                         // row r: w[2 r], columns 4 part .. and w[2 r + 1], 32 further on, so that a load reads whole lines
    uint32_t size[8];
    __device__ __forceinline__ static int column(int part, int c) { return 4 * part + (c & 3) + (c >> 2) * 32; }
    __device__ __forceinline__ uint32_t bits(int r, int c) const { return uint32_t(w[2 * r + c / 4][c % 4]); }
    __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
    __device__ __forceinline__ void sizes() {
        uint32_t all = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            size[c] = 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) size[c] = larger(size[c], bits(r, c) & 0x7fffffffu);
            all = larger(all, size[c]);
        }
        if (__any(all >= 0x7f800000u)) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                size[c] = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t b = bits(r, c) & 0x7fffffffu;
                    size[c] = larger(size[c], b >= 0x7f800000u ? 0u : b);
                }
            }
        }
    }
    static constexpr int SIZES = 8;
    __device__ __forceinline__ uint32_t& size_at(int i) { return size[i]; }
    __device__ __forceinline__ static uint32_t size_in(const uint32_t* sizes, int j) { return sizes[(j & 31) / 4 * 8 + (j & 3) + j / 32 * 4]; }
    __device__ __forceinline__ static int exponent_of(uint32_t size) { return int((larger(size, 0x0d800000u) + 0x1fffffu) >> 23) - 8; }
    __device__ __forceinline__ int exponent(int c) const { return exponent_of(size[c]); }
    __device__ __forceinline__ int codes(int c, int e) const {
        typedef short i16x2 __attribute__((ext_vector_type(2)));
        const float scale = __builtin_bit_cast(float, e << 23);
        i16x2 q{0, 0};
        q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q, __builtin_bit_cast(float, bits(0, c)), __builtin_bit_cast(float, bits(1, c)), scale, false);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q, __builtin_bit_cast(float, bits(2, c)), __builtin_bit_cast(float, bits(3, c)), scale, true);
        return __builtin_bit_cast(int, q);
    }
};

// by_columns: all K blocks of a column tile run on one XCD, where enough of them are for all eight: its L2 then holds the tile's columns, and neighbouring
// K blocks' lines are written at about the same time (fp32 4096 x 4096 gathered four times over 47.8 -> 39.5 us, bf16 4096 x 7168 19.2 -> 17.8 gathered once,
// 21.9 -> 21.1 as it is). PAST: codes of more than 64 MB of rows gathered twice or more are stored past the caches, which plain stores push the source out of
// (bf16, gathered four times: 4096 x 7168 55.0 -> 31.1 us, 8192 x 4096 66.5 -> 37.5; fp32 4096 x 4096 gathered eight times 71 -> 44). The product behind reads
// them from further away: both together 665 -> 651 and 344 -> 340 us; below 64 MB, or as they are, they would lose 1 to 5 % (2048 x 2048 x 8 88.7 -> 93.0).
template <typename T, bool GATHER, bool STREAM, bool PAST>
__global__ void __launch_bounds__(256)
per_channel_cast_kernel(const T* __restrict__ x, const int* __restrict__ source, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                        int m, int n, int k_blocks, int scales_stride, int column_tiles, bool by_columns) {
    using Tile = CastTile<sizeof(T)>;
    constexpr int PITCH = 136;          // bytes between the columns in LDS: whole 8 bytes, and 64 lanes' dwords over the banks twice at most
    constexpr int SIZES = Tile::SIZES, PIECES = sizeof(T) / 2;
    __shared__ __attribute__((aligned(16))) uint32_t wave_size[4][8][SIZES];
    __shared__ __attribute__((aligned(16))) uint8_t turned[kCastColumns * PITCH];
    int kb, column_tile;
    if (by_columns) {
        const int i = int(blockIdx.x) / kNumXCD;
        column_tile = i / k_blocks * kNumXCD + int(blockIdx.x) % kNumXCD;
        kb = i % k_blocks;
        if (column_tile >= column_tiles) return;
    } else {
        kb = int(blockIdx.x) / column_tiles;
        column_tile = int(blockIdx.x) - kb * column_tiles;
    }
    const int j0 = column_tile * kCastColumns;
    const int part = threadIdx.x & 7, quad = threadIdx.x >> 3, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile tile;
    i32x4 rows;
    if constexpr (GATHER) rows = *reinterpret_cast<const i32x4*>(source + kb * 128 + quad * 4);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = GATHER ? rows[r] : kb * 128 + quad * 4 + r;
        const bool live = uint32_t(row) < uint32_t(m);
        const T* const from = x + size_t(live ? row : 0) * n + j0;
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
            tile.w[PIECES * r + h] = i32x4{0, 0, 0, 0};
            const int column = Tile::column(part, 4 * h);
            if (live && j0 + column < n) {
                const i32x4* piece = reinterpret_cast<const i32x4*>(from + column);
                tile.w[PIECES * r + h] = STREAM ? __builtin_nontemporal_load(piece) : *piece;
            }
        }
    }
    // the columns' sizes: this thread's rows, the eight threads of the wave that have the same columns, the four waves
    tile.sizes();
#pragma unroll
    for (int i = 0; i < SIZES; ++i) {
        uint32_t a = tile.size_at(i);
        a = Tile::larger(a, uint32_t(__builtin_amdgcn_update_dpp(0, int(a), 0x128, 0xf, 0xf, true)));         // rotated by 8 in the 16 lanes
        auto pair = __builtin_amdgcn_permlane16_swap(a, a, false, false);
        a = Tile::larger(pair[0], pair[1]);
        pair = __builtin_amdgcn_permlane32_swap(a, a, false, false);
        a = Tile::larger(pair[0], pair[1]);
        tile.size_at(i) = a;
    }
    if (lane < 8) {
#pragma unroll
        for (int i = 0; i < SIZES; ++i) wave_size[wave][part][i] = tile.size_at(i);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SIZES; ++i)
        tile.size_at(i) = Tile::larger(Tile::larger(wave_size[0][part][i], wave_size[1][part][i]), Tile::larger(wave_size[2][part][i], wave_size[3][part][i]));
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        *reinterpret_cast<int*>(turned + Tile::column(part, c) * PITCH + quad * 4) = tile.codes(c, tile.exponent(c));         // (19 to 247)
    }
    if (wave == 3 && j0 + lane < n) {           // a lane a column
        const auto size_of = [&](int w) { return Tile::size_in(&wave_size[w][0][0], lane); };
        const uint32_t size = max(max(size_of(0), size_of(1)), max(size_of(2), size_of(3)));
        scales[size_t(j0 + lane) * scales_stride + kb] = uint8_t(Tile::exponent_of(size));
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int column = p * 32 + quad;
        if (j0 + column >= n) continue;
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 lo = *reinterpret_cast<const u32x2*>(turned + column * PITCH + part * 16), hi = *reinterpret_cast<const u32x2*>(turned + column * PITCH + part * 16 + 8);
        const i32x4 v = i32x4{int(lo[0]), int(lo[1]), int(hi[0]), int(hi[1])};
        i32x4* const to = reinterpret_cast<i32x4*>(codes + (size_t(j0 + column) * k_blocks + kb) * 128 + part * 16);
        if constexpr (PAST) __builtin_nontemporal_store(v, to);
        else *to = v;
    }
}

// x [m, n] row-major, n % 8 == 0, 16-byte aligned -> codes [n, 128 k_blocks], scales byte (j, b) at j * scales_stride + b. `source`: [128 k_blocks] or null.
template <typename T>
inline hipError_t launch_per_channel_cast(const T* x, const int* source, void* codes, uint8_t* scales, int m, int n, int k_blocks, int scales_stride,
                                          hipStream_t stream) {
    if (m < 0 || n < 0 || n % 8 != 0 || k_blocks < 0 || scales_stride < k_blocks) return hipErrorInvalidValue;
    if (n == 0 || k_blocks == 0) return hipSuccess;
    if ((m && !x) || !codes || !scales || (!source && ceil_div(m, 128) > k_blocks)) return hipErrorInvalidValue;
    const int column_tiles = ceil_div(n, kCastColumns);
    const bool by_columns = column_tiles % kNumXCD == 0 || column_tiles >= 4 * kNumXCD;
    const long long blocks = (long long)(by_columns ? ceil_div(column_tiles, kNumXCD) * kNumXCD : column_tiles) * k_blocks;
    if (blocks >= 1ll << 24) return hipErrorInvalidValue;         // a launch has less than 2^32 threads
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(uint32_t(blocks)), dim3(256), 0, stream, x, source, static_cast<uint8_t*>(codes), scales, m, n, k_blocks, scales_stride, column_tiles, by_columns);
        return hipGetLastError();
    };
    if (source) {
        // a source whose rows are read over and over stays in the L2s if the codes go past them
        const bool past = (long long)n * k_blocks * 128 > kCastPastBytes && 128ll * k_blocks >= 2ll * m;
        return past ? launch(per_channel_cast_kernel<T, true, false, true>) : launch(per_channel_cast_kernel<T, true, false, false>);
    }
    return (long long)m * n * (long long)sizeof(T) > kCastL2Bytes ? launch(per_channel_cast_kernel<T, false, true, false>) : launch(per_channel_cast_kernel<T, false, false, false>);
}

} // namespace yan
