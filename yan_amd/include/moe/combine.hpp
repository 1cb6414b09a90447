// The experts' outputs back to their tokens, and the gradients of that.
//
//   out[t] = sum_i w[t, i] y[rows[t, i]], in fp32, rounded to bf16 once; a pair without a row (negative, or from M on) adds nothing
//   backward, from dout: dy[rows[t, i]] = w[t, i] dout[t], rows that no pair has become zero; dw[t, i] = <dout[t], y[rows[t, i]]>
//
// Bound by HBM: the forward reads top_k rows a token and writes one; the backward reads the rows again and writes all of dy.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <algorithm>

#include "lanes.hpp"
#include "route.hpp"

namespace yan {

__device__ __forceinline__ void bf16x8_to_float(float (&f)[8], i32x4 raw) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __builtin_bit_cast(float, uint32_t(raw[i]) << 16);
        f[2 * i + 1] = __builtin_bit_cast(float, uint32_t(raw[i]) & 0xffff0000u);
    }
}
__device__ __forceinline__ i32x4 float_to_bf16x8(const float (&f)[8]) {
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<__bf16>(f[i]);
    return __builtin_bit_cast(i32x4, v);
}

// A wave has 512 columns of a token, a lane eight of them, so that rows and weights are the wave's own and come by scalar loads. rows_of / weights:
// [tokens, TOP_K]; weights may be null (all 1).
template <int TOP_K>
__global__ void __launch_bounds__(256)
moe_combine_kernel(const __bf16* __restrict__ y, const int* __restrict__ rows_of, const float* __restrict__ weights, __bf16* __restrict__ out,
                   int tokens, int pieces, int rows, int waves_per_token) {
    const long long unit = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
    const int t = int(unit / waves_per_token), c = int(unit - (long long)t * waves_per_token) * kWaveSize + int(threadIdx.x % kWaveSize);
    if (t >= tokens) return;
    if (c >= pieces) return;
    i32x4 raw[TOP_K];
    float w[TOP_K];
    bool live[TOP_K];
#pragma unroll
    for (int i = 0; i < TOP_K; ++i) {           // without branches between the loads: a pair without a row reads row 0 and forgets it
        const int row = rows_of[size_t(t) * TOP_K + i];
        live[i] = uint32_t(row) < uint32_t(rows);
        w[i] = weights ? weights[size_t(t) * TOP_K + i] : 1.f;
        raw[i] = i32x4{0, 0, 0, 0};
        if (rows) raw[i] = reinterpret_cast<const i32x4*>(y)[size_t(live[i] ? row : 0) * pieces + c];
    }
#pragma unroll
    for (int i = 0; i < TOP_K; ++i)
        if (!live[i]) w[i] = 0.f, raw[i] = i32x4{0, 0, 0, 0};
    float sum[8] = {};
#pragma unroll
    for (int i = 0; i < TOP_K; ++i) {
        float f[8];
        bf16x8_to_float(f, raw[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = fmaf(w[i], f[j], sum[j]);
    }
    reinterpret_cast<i32x4*>(out)[size_t(t) * pieces + c] = float_to_bf16x8(sum);
}

// THREADS a token, 256 / THREADS tokens a workgroup; the workgroups from `token_blocks` on clear the rows that no pair has. A wave a token only where it
// holds all of the columns (1024 columns, 4000 x 8 pairs, forward and backward: 55.0 us with a wave a token, 35.1 with a workgroup). STREAM: y is read for the
// last time and dy outgrows the L2s by so much that both go past them; forward and backward of tokens x 8 x 4096, plain / so: 4097 (300 MB of dy)
// 231.7 / 208.9 us, 2048 117.0 / 110.7, 1024 65.0 / 61.8, 512 34.7 / 37.1.
constexpr long long kCombineStreamBytes = 64ll << 20;
constexpr int kRowsPerClearBlock = 32;
template <int TOP_K, int THREADS, bool STREAM>
__global__ void __launch_bounds__(256)
moe_combine_backward_kernel(const __bf16* __restrict__ grad_out, const __bf16* __restrict__ y, const int* __restrict__ rows_of,
                            const float* __restrict__ weights, const int* __restrict__ source, __bf16* __restrict__ grad_y, float* __restrict__ grad_weights,
                            int tokens, int pieces, int rows, int token_blocks) {
    __shared__ float parts[4][TOP_K];
    if (int(blockIdx.x) >= token_blocks) {
        const int first = (int(blockIdx.x) - token_blocks) * kRowsPerClearBlock;
        for (int r = first + int(threadIdx.x >> 6); r < min(rows, first + kRowsPerClearBlock); r += 4) {
            if (source[r] >= 0) continue;
            for (int c = threadIdx.x & 63; c < pieces; c += 64) reinterpret_cast<i32x4*>(grad_y)[size_t(r) * pieces + c] = i32x4{0, 0, 0, 0};
        }
        return;
    }
    const int t = blockIdx.x * (256 / THREADS) + int(threadIdx.x) / THREADS;
    const bool live = t < tokens;
    int row[TOP_K];
    float w[TOP_K], dot[TOP_K];
#pragma unroll
    for (int i = 0; i < TOP_K; ++i) {
        row[i] = live ? rows_of[size_t(t) * TOP_K + i] : -1;
        if (uint32_t(row[i]) >= uint32_t(rows)) row[i] = -1;
        w[i] = weights && live ? weights[size_t(t) * TOP_K + i] : 1.f;
        dot[i] = 0.f;
    }
    if (live) {
        for (int c = threadIdx.x % THREADS; c < pieces; c += THREADS) {
            float d[8];
            bf16x8_to_float(d, reinterpret_cast<const i32x4*>(grad_out)[size_t(t) * pieces + c]);
            i32x4 raw[TOP_K];
            if (grad_weights) {
#pragma unroll
                for (int i = 0; i < TOP_K; ++i) {
                    raw[i] = i32x4{0, 0, 0, 0};
                    const i32x4* const from = reinterpret_cast<const i32x4*>(y) + size_t(row[i]) * pieces + c;
                    if (row[i] >= 0) raw[i] = STREAM ? __builtin_nontemporal_load(from) : *from;
                }
            }
#pragma unroll
            for (int i = 0; i < TOP_K; ++i) {
                if (row[i] < 0) continue;
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = w[i] * d[j];
                i32x4* const to = reinterpret_cast<i32x4*>(grad_y) + size_t(row[i]) * pieces + c;
                if (STREAM) __builtin_nontemporal_store(float_to_bf16x8(f), to);
                else *to = float_to_bf16x8(f);
                if (grad_weights) {
                    bf16x8_to_float(f, raw[i]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) dot[i] = fmaf(d[j], f[j], dot[i]);
                }
            }
        }
    }
    if (!grad_weights) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < TOP_K; ++i) {
        dot[i] = sum_lanes<64>(dot[i]);
        if constexpr (THREADS == 64) {
            if (live && lane == 0) grad_weights[size_t(t) * TOP_K + i] = dot[i];
        } else if (lane == 0) {
            parts[wave][i] = dot[i];
        }
    }
    if constexpr (THREADS == 256) {
        __syncthreads();
        if (threadIdx.x < TOP_K) grad_weights[size_t(t) * TOP_K + threadIdx.x] = (parts[0][threadIdx.x] + parts[1][threadIdx.x]) + (parts[2][threadIdx.x] + parts[3][threadIdx.x]);
    }
}

// y [rows, columns], columns % 8 == 0, both 16-byte aligned
template <int TOP_K>
inline hipError_t launch_moe_combine(const __bf16* y, const int* rows_of, const float* weights, __bf16* out, int tokens, int columns, int rows, hipStream_t stream) {
    if (tokens < 0 || tokens > kMaxTokens || columns < 0 || columns % 8 != 0 || rows < 0) return hipErrorInvalidValue;
    if (tokens == 0 || columns == 0) return hipSuccess;
    if (!rows_of || !out || (rows && !y)) return hipErrorInvalidValue;
    const int pieces = columns / 8;
    const int waves_per_token = ceil_div(pieces, kWaveSize);
    const long long blocks = ceil_div((long long)tokens * waves_per_token, 4ll);
    if (blocks > kMaxWorkgroups) return hipErrorInvalidValue;
    hipLaunchKernelGGL(moe_combine_kernel<TOP_K>, dim3(uint32_t(blocks)), dim3(256), 0, stream, y, rows_of, weights, out, tokens, pieces, rows, waves_per_token);
    return hipGetLastError();
}

template <int TOP_K>
inline hipError_t launch_moe_combine_backward(const __bf16* grad_out, const __bf16* y, const int* rows_of, const float* weights, const int* source,
                                              __bf16* grad_y, float* grad_weights, int tokens, int columns, int rows, hipStream_t stream) {
    if (tokens < 0 || tokens > kMaxTokens || columns < 0 || columns % 8 != 0 || rows < 0) return hipErrorInvalidValue;
    // (without columns there is nothing behind y and the gradients, and the weights' gradient is zero)
    if (tokens && (!rows_of || (columns && !grad_out))) return hipErrorInvalidValue;
    if (rows && (!source || (columns && (!grad_y || !y)))) return hipErrorInvalidValue;
    const int pieces = columns / 8;
    const bool wide = pieces > kWaveSize;
    const int token_blocks = wide ? tokens : ceil_div(tokens, 4), clear_blocks = ceil_div(rows, kRowsPerClearBlock);
    if ((long long)token_blocks + clear_blocks > kMaxWorkgroups) return hipErrorInvalidValue;
    if (token_blocks + clear_blocks == 0) return hipSuccess;
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(token_blocks + clear_blocks), dim3(256), 0, stream, grad_out, y, rows_of, weights, source, grad_y, grad_weights, tokens,
                           pieces, rows, token_blocks);
        return hipGetLastError();
    };
    if (!wide) return launch(moe_combine_backward_kernel<TOP_K, 64, false>);
    return (long long)rows * columns * 2 > kCombineStreamBytes ? launch(moe_combine_backward_kernel<TOP_K, 256, true>)
                                                               : launch(moe_combine_backward_kernel<TOP_K, 256, false>);
}

} // namespace yan
