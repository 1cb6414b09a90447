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
constexpr float kLeastAmax = 0x1p-100f;

// e + 127 of the smallest e with amax <= 448 * 2^e; amax is a normal number. 448 = 1.75 * 2^8.
__device__ __forceinline__ int exponent_for(float amax) {
    const int bits = __builtin_bit_cast(int, amax);
    return (bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
}

// Four rows of eight columns as loaded.
template <typename T> struct Raw4x8 { i32x4 w[4][sizeof(T) / 2]; };

// Taking four K blocks a workgroup, the next one's rows under way during the one before, or all K blocks of a column tile on one XCD, whose L2 then holds
// the tile's columns, was no faster (4096 x 7168 gathered four times over: 68.0 us as it is, 70.2, 71.6).
template <typename T, bool GATHER, bool STREAM>
__global__ void __launch_bounds__(256)
per_channel_cast_kernel(const T* __restrict__ x, const int* __restrict__ source, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                        int m, int n, int k_blocks, int scales_stride, int column_tiles) {
    constexpr int PITCH = 136;          // bytes between the columns in LDS: whole 8 bytes, and 64 lanes' dwords over the banks twice at most
    __shared__ float wave_max[4][kCastColumns];
    __shared__ __attribute__((aligned(16))) uint8_t turned[kCastColumns * PITCH];
    const int kb = int(blockIdx.x) / column_tiles, j0 = (int(blockIdx.x) - kb * column_tiles) * kCastColumns;
    const int part = threadIdx.x & 7, quad = threadIdx.x >> 3, wave = threadIdx.x >> 6;
    // element c of this thread's eight is column 8 part + c of bf16; of fp32 4 part + c and 32 further on, so that a load reads whole lines
    const auto column_of = [&](int c) { return sizeof(T) == 2 ? 8 * part + c : 4 * part + (c & 3) + (c >> 2) * 32; };
    Raw4x8<T> raw;
    i32x4 rows;
    if constexpr (GATHER) rows = *reinterpret_cast<const i32x4*>(source + kb * 128 + quad * 4);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = GATHER ? rows[r] : kb * 128 + quad * 4 + r;
        const bool live = uint32_t(row) < uint32_t(m);
#pragma unroll
        for (int h = 0; h < int(sizeof(T) / 2); ++h) {
            raw.w[r][h] = i32x4{0, 0, 0, 0};
            const int column = j0 + column_of(4 * h);
            if (live && column < n) {
                const i32x4* from = reinterpret_cast<const i32x4*>(x + size_t(row) * n + column);
                raw.w[r][h] = STREAM ? __builtin_nontemporal_load(from) : *from;
            }
        }
    }
    float v[4][8];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            uint32_t bits;
            if constexpr (sizeof(T) == 4) bits = uint32_t(raw.w[r][c / 4][c % 4]);
            else bits = c % 2 ? uint32_t(raw.w[r][0][c / 2]) & 0xffff0000u : uint32_t(raw.w[r][0][c / 2]) << 16;
            v[r][c] = __builtin_bit_cast(float, bits);
        }
    // the columns' maxima: this thread's rows, the eight threads of the wave that have the same columns, the four waves
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        float a = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float size = fabsf(v[r][c]);
            a = fmaxf(a, size < __builtin_inff() ? size : 0.f);
        }
        a = fmaxf(a, rotate_in_16_lanes<8>(a));
        auto pair = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, a), false, false);
        a = fmaxf(__builtin_bit_cast(float, uint32_t(pair[0])), __builtin_bit_cast(float, uint32_t(pair[1])));
        pair = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, a), false, false);
        a = fmaxf(__builtin_bit_cast(float, uint32_t(pair[0])), __builtin_bit_cast(float, uint32_t(pair[1])));
        if ((threadIdx.x & 63) < 8) wave_max[wave][column_of(c)] = a;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const int column = column_of(c);
        const float amax = fmaxf(fmaxf(fmaxf(wave_max[0][column], wave_max[1][column]), fmaxf(wave_max[2][column], wave_max[3][column])), kLeastAmax);
        const int e = exponent_for(amax);
        const float factor = __builtin_bit_cast(float, (254 - e) << 23);         // 2^-(e - 127); e is 19 to 247
        if (quad == 0 && j0 + column < n) scales[size_t(j0 + column) * scales_stride + kb] = uint8_t(e);
        int q = 0;
        q = __builtin_amdgcn_cvt_pk_fp8_f32(v[0][c] * factor, v[1][c] * factor, q, false);
        q = __builtin_amdgcn_cvt_pk_fp8_f32(v[2][c] * factor, v[3][c] * factor, q, true);
        *reinterpret_cast<int*>(turned + column * PITCH + quad * 4) = q;
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int column = p * 32 + quad;
        if (j0 + column >= n) continue;
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 lo = *reinterpret_cast<const u32x2*>(turned + column * PITCH + part * 16), hi = *reinterpret_cast<const u32x2*>(turned + column * PITCH + part * 16 + 8);
        *reinterpret_cast<i32x4*>(codes + (size_t(j0 + column) * k_blocks + kb) * 128 + part * 16) = i32x4{int(lo[0]), int(lo[1]), int(hi[0]), int(hi[1])};
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
    const long long blocks = (long long)column_tiles * k_blocks;
    if (blocks >= 1ll << 31) return hipErrorInvalidValue;
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(uint32_t(blocks)), dim3(256), 0, stream, x, source, static_cast<uint8_t*>(codes), scales, m, n, k_blocks, scales_stride, column_tiles);
        return hipGetLastError();
    };
    if (source) return launch(per_channel_cast_kernel<T, true, false>);
    return (long long)m * n * (long long)sizeof(T) > kCastL2Bytes ? launch(per_channel_cast_kernel<T, false, true>) : launch(per_channel_cast_kernel<T, false, false>);
}

} // namespace yan
