// Root-mean-square norm with the addition of the residual in front of it and the quantiser of the FP8 GEMMs behind it, and its gradient.
//
//   h = T(x + residual), which replaces the residual (without one h = x);   r = (sum h^2 / k + eps)^-1/2;   y = (h r) w
//   normed = bf16(y);   codes, scales: y quantised 1 x 128 with the arithmetic of per_token_cast_kernel, from the fp32 y
//   backward:  u = h r,  p = g w:   dh = r (p - u sum(p u) / k) + grad_residual;   dw = sum over the rows of g u
// Squares, products and the sums over rows are fp32; the only roundings are h to the residual's type, which is what the next layer reads, and the outputs'.
//
// Bound by HBM. A row lies in the registers of LANES lanes from its load to its last store, V runs of 8 elements a lane, lane l of run v with elements
// 8 (v LANES + l) .. + 7, so that 16 neighbouring lanes have the 128 elements of a scale and every load covers whole lines. One pass: separate kernels for
// addition, norm and quantiser would move the row four times more. 8192 x 7168, bf16, a residual, codes and 16 bits (530 MB): 108 us, 4.9 TB/s, where a large copy has 5.1;
// 64 x 7168: 3.8 us, a launch's latency and two trips to memory.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "../gemm/fp8_cast.hpp"
#include "../moe/lanes.hpp"

namespace yan {

constexpr int kNormMostColumns = 16384;         // forward 256 lanes with eight runs each, backward 1024 with two

// Eight elements from `p` on, as loaded.
template <typename T>
__device__ __forceinline__ Raw8<T> load_run(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const i32x4*>(p)[i];
    return r;
}

// Eight numbers rounded to T.
template <typename T>
__device__ __forceinline__ Raw8<T> round_run(const F32x8& f) {
    Raw8<T> r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i / 4][i % 4] = __builtin_bit_cast(int, f.v[i]);
    } else {
        bf16x8 b;
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = __bf16(f.v[i]);
        r.w[0] = __builtin_bit_cast(i32x4, b);
    }
    return r;
}
// To `p` on.
template <typename T>
__device__ __forceinline__ void store_run(T* p, const Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) reinterpret_cast<i32x4*>(p)[i] = r.w[i];
}

// What was made of `r` before this is made of it again behind it, not kept.
template <typename T>
__device__ __forceinline__ void make_anew(Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) asm volatile("" : "+v"(r.w[i]));
}

// The sum over the LANES lanes of a row, the same in all of them. Up to a wave in registers; more lanes are the whole workgroup, whose waves leave their sums in
// `slots`, which the next call may not be given again.
template <int LANES>
__device__ __forceinline__ float sum_row(float v, float* slots) {
    if constexpr (LANES <= 64) {
        return sum_lanes<LANES>(v);
    } else {
        constexpr int WAVES = LANES / kWaveSize;
        v = sum_lanes<64>(v);
        if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
        __syncthreads();
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += slots[w];
        return sum;
    }
}

struct NormShape {
    int rows, k;
    float eps;
    long long stride_m, stride_k;           // of the scales, in elements
};

// Neighbouring rows run on one XCD at about the same time: token-contiguous scales of a K block are 4 bytes from each of them, and come together to lines in its L2.
__device__ __forceinline__ int norm_block_of(int bid, int blocks) {
    const int per_xcd = ceil_div(blocks, kNumXCD);
    return bid % kNumXCD * per_xcd + bid / kNumXCD;
}

// Rows are taken ROWS at a time, by groups of lanes: how many times that is, whether row `group` of number `block` exists, and which it is, the last one where it does not. (No number here
// passes the last row's, which may be the largest of 31 bits.)
template <int ROWS> __host__ __device__ __forceinline__ int norm_blocks(int rows) { return rows / ROWS + (rows % ROWS != 0); }
template <int ROWS> __host__ __device__ __forceinline__ bool norm_row_exists(int block, int group, int rows) { return group < rows - block * ROWS; }
template <int ROWS> __host__ __device__ __forceinline__ int norm_row(int block, int group, int rows) {
    return norm_row_exists<ROWS>(block, group, rows) ? block * ROWS + group : rows - 1;
}

// residual (RESIDUAL) is h's place too; codes and scales if CODES, normed if NORMED. `out` may be x.
template <typename X, typename H, typename W, int LANES, int V, bool RESIDUAL, bool CODES, bool NORMED>
__global__ void __launch_bounds__(LANES > 256 ? LANES : 256)
rms_norm_kernel(const X* x, H* residual, const W* __restrict__ weight, uint8_t* __restrict__ codes, float* __restrict__ scales, __bf16* normed,
                float* __restrict__ inverse_rms, NormShape s) {
    constexpr int THREADS = LANES > 256 ? LANES : 256, ROWS = THREADS / LANES;
    __shared__ float slots[LANES > 64 ? LANES / kWaveSize : 1];
    const int lane = threadIdx.x % LANES, blocks = norm_blocks<ROWS>(s.rows), block = norm_block_of(blockIdx.x, blocks);
    if (block >= blocks) return;
    // (rows behind the last one are read and reduced in its place, since all lanes of a wave have to take part, and not stored)
    const int row = norm_row<ROWS>(block, threadIdx.x / LANES, s.rows);
    const bool live = norm_row_exists<ROWS>(block, threadIdx.x / LANES, s.rows);
    const size_t at = size_t(row) * s.k;
    F32x8 h[V];
    Raw8<X> raw[V];
    Raw8<H> old[RESIDUAL ? V : 1];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * LANES + lane) * 8;
        raw[v] = Raw8<X>{};
        if constexpr (RESIDUAL) old[v] = Raw8<H>{};
        if (c < s.k) {
            raw[v] = load_run(x + at + c);
            if constexpr (RESIDUAL) old[v] = load_run(residual + at + c);
        }
    }
    Raw8<W> w[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * LANES + lane) * 8;
        w[v] = Raw8<W>{};
        if (c < s.k) w[v] = load_run(weight + c);
    }
    float square = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * LANES + lane) * 8;
        h[v] = to_f32(raw[v]);
        if constexpr (RESIDUAL) {
            const F32x8 before = to_f32(old[v]);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[v].v[i] += before.v[i];
            const Raw8<H> sum = round_run<H>(h[v]);
            if (live && c < s.k) store_run(residual + at + c, sum);
            h[v] = to_f32(sum);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) square = fmaf(h[v].v[i], h[v].v[i], square);
    }
    const float inverse = 1.f / sqrtf(sum_row<LANES>(square, slots) / float(s.k) + s.eps);
    if (live && lane == 0) inverse_rms[row] = inverse;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * LANES + lane) * 8;
        const F32x8 by = to_f32(w[v]);
        F32x8 y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y.v[i] = h[v].v[i] * inverse * by.v[i];
        if constexpr (NORMED) {
            if (live && c < s.k) store_run(normed + at + c, round_run<__bf16>(y));
        }
        if constexpr (CODES) {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            const float amax = fmaxf(max_over_16_lanes(abs_max8(y)), 1e-4f);
            const uint2 q = quantise8(y, kFp8Max / amax);
            if (live && c < s.k) {
                *reinterpret_cast<u32x2*>(codes + at + c) = u32x2{q.x, q.y};
                if (lane % 16 == 0) scales[row * s.stride_m + c / 128 * s.stride_k] = amax / kFp8Max;
            }
        }
    }
}

// A workgroup takes rows blockIdx.x, + gridDim.x, ... (groups of THREADS / LANES of them), the next one's loads under way while it adds up; each lane keeps the
// weight's sums of its columns and leaves them in row blockIdx.x * ROWS + its group of `partial` [parts, k] (WEIGHT). Adding to the gradient itself by atomics would
// save the second launch and make results differ from run to run; a meeting of the workgroups, whose last adds up in order, would not, and has not been built. 8192 x 7168 with a residual's gradient (470 MB): 93 us with the sums, 5.1 TB/s.
template <typename G, typename H, typename W, int LANES, int V, bool RESIDUAL, bool WEIGHT>
__global__ void __launch_bounds__(LANES > 256 ? LANES : 256)
rms_norm_backward_kernel(const G* __restrict__ grad, const H* __restrict__ h, const W* __restrict__ weight, const float* __restrict__ inverse_rms,
                         const G* __restrict__ grad_residual, G* __restrict__ grad_h, float* __restrict__ partial, int rows, int k) {
    constexpr int THREADS = LANES > 256 ? LANES : 256, ROWS = THREADS / LANES, WAVES = LANES > 64 ? LANES / kWaveSize : 1;
    __shared__ float slots[2][WAVES];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, blocks = norm_blocks<ROWS>(rows);
    Raw8<W> w[V];
    F32x8 sums[WEIGHT ? V : 1];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * LANES + lane) * 8;
        w[v] = Raw8<W>{};
        if (c < k) w[v] = load_run(weight + c);
        if constexpr (WEIGHT) sums[v] = F32x8{};
    }
    struct Row {
        Raw8<G> g[V], kept[RESIDUAL ? V : 1];
        Raw8<H> h[V];
        float inverse;
    };
    const auto load = [&](Row& r, int block) __attribute__((always_inline)) {
        const int row = norm_row<ROWS>(block, group, rows);
        const size_t at = size_t(row) * k;
        r.inverse = inverse_rms[row];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * LANES + lane) * 8;
            r.g[v] = Raw8<G>{};
            r.h[v] = Raw8<H>{};
            if constexpr (RESIDUAL) r.kept[v] = Raw8<G>{};
            if (c < k) {
                r.g[v] = load_run(grad + at + c);
                r.h[v] = load_run(h + at + c);
                if constexpr (RESIDUAL) r.kept[v] = load_run(grad_residual + at + c);
            }
        }
    };
    const auto step = [&](Row& r, int block, int turn) __attribute__((always_inline)) {
        const size_t at = size_t(norm_row<ROWS>(block, group, rows)) * k;
        const bool live = norm_row_exists<ROWS>(block, group, rows);
        float dot = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const F32x8 g = to_f32(r.g[v]), x = to_f32(r.h[v]), by = to_f32(w[v]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = x.v[i] * r.inverse;
                dot = fmaf(g.v[i] * by.v[i], u, dot);
                if constexpr (WEIGHT) {
                    if (live) sums[v].v[i] = fmaf(g.v[i], u, sums[v].v[i]);
                }
            }
        }
        dot = sum_row<LANES>(dot, slots[turn]) / float(k);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * LANES + lane) * 8;
            if constexpr (LANES > 256) make_anew(r.g[v]), make_anew(r.h[v]), make_anew(w[v]);
            const F32x8 g = to_f32(r.g[v]), x = to_f32(r.h[v]), by = to_f32(w[v]);
            F32x8 down;
#pragma unroll
            for (int i = 0; i < 8; ++i) down.v[i] = r.inverse * (g.v[i] * by.v[i] - x.v[i] * r.inverse * dot);
            if constexpr (RESIDUAL) {
                const F32x8 kept = to_f32(r.kept[v]);
#pragma unroll
                for (int i = 0; i < 8; ++i) down.v[i] += kept.v[i];
            }
            if (live && c < k) store_run(grad_h + at + c, round_run<G>(down));
        }
    };
    int block = blockIdx.x;
    if constexpr (LANES <= 256) {
        Row a, b;
        if (block < blocks) load(a, block);
        // (two rows a turn, each in registers and slots of its own)
        while (block < blocks) {
            const int second = block + gridDim.x, third = second + gridDim.x;
            if (second < blocks) load(b, second);
            step(a, block, 0);
            if (second < blocks) {
                if (third < blocks) load(a, third);
                step(b, second, 1);
            }
            block = third;
        }
    } else {
        // Wider rows, of 1024 lanes, have no registers for a second one. The loads of sixteen waves, and the stores of the row before, hide each other well enough: 8192 x 16384, bf16, with a
        // residual's gradient (1.07 GB): 200 us, 5.4 TB/s. Everything stays in registers but for 20 bytes of a lane where h and the weight are fp32 and both the residual's gradient and
        // the weight's are asked for.
        Row a;
        for (int turn = 0; block < blocks; block += gridDim.x, turn ^= 1) {
            load(a, block);
            step(a, block, turn);
        }
    }
    if constexpr (WEIGHT) {
        float* const to = partial + (size_t(blockIdx.x) * ROWS + group) * k;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * LANES + lane) * 8;
            if (c < k) {
                *reinterpret_cast<f32x4*>(to + c) = f32x4{sums[v].v[0], sums[v].v[1], sums[v].v[2], sums[v].v[3]};
                *reinterpret_cast<f32x4*>(to + c + 4) = f32x4{sums[v].v[4], sums[v].v[5], sums[v].v[6], sums[v].v[7]};
            }
        }
    }
}

// out [k] (+)= the sum of the `parts` rows of `partial`, in a fixed order: 32 columns a workgroup, 32 threads a column, each with every 32nd row.
template <int = 0>
__global__ void __launch_bounds__(1024)
rms_norm_weight_sum_kernel(const float* __restrict__ partial, float* __restrict__ out, int parts, int k, bool accumulate) {
    __shared__ float sums[32][33];
    const int column = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + column;
    float sum = 0.f;
    if (c < k) {
#pragma unroll 8
        for (int p = part; p < parts; p += 32) sum += partial[size_t(p) * k + c];
    }
    sums[part][column] = sum;
    __syncthreads();
    if (part == 0 && c < k) {
        float total = accumulate ? out[c] : 0.f;
#pragma unroll
        for (int p = 0; p < 32; ++p) total += sums[p][column];
        out[c] = total;
    }
}

// Rows of the norm that one launch takes: whole rounds of workgroups over the XCDs.
constexpr int norm_rows_per_launch(int threads, int rows) { return int(((1ll << 32) / threads - 1) / kNumXCD * kNumXCD * rows); }

// x [rows, k]; residual null where !RESIDUAL; scales [rows, k / 128] with the strides given.
template <typename X, typename H, typename W, int LANES, int V, bool RESIDUAL, bool CODES, bool NORMED>
inline hipError_t launch_rms_norm(const X* x, H* residual, const W* weight, void* codes, float* scales, long long stride_m, long long stride_k, void* normed,
                                  float* inverse_rms, int rows, int k, float eps, hipStream_t stream) {
    static_assert(CODES || NORMED);
    if (rows < 0 || k <= 0 || k > kNormMostColumns || k % (CODES ? 128 : 8) != 0 || k > LANES * V * 8 || stride_m < 0 || stride_k < 0) return hipErrorInvalidValue;
    if (rows == 0) return hipSuccess;
    if (!x || !weight || !inverse_rms || (RESIDUAL && !residual) || (CODES && (!codes || !scales)) || (NORMED && !normed)) return hipErrorInvalidValue;
    constexpr int THREADS = LANES > 256 ? LANES : 256, ROWS = THREADS / LANES;
    // A launch has less than 2^32 threads; more rows than those have, from 2^24 of 256 lanes and 2^28 of 16 on, are several launches.
    constexpr int MOST = norm_rows_per_launch(THREADS, ROWS);
    for (long long first = 0; first < rows; first += MOST) {
        const int here = int(std::min<long long>(MOST, rows - first));
        const size_t at = size_t(first) * k;
        hipLaunchKernelGGL((rms_norm_kernel<X, H, W, LANES, V, RESIDUAL, CODES, NORMED>), dim3(ceil_div(norm_blocks<ROWS>(here), kNumXCD) * kNumXCD), dim3(THREADS), 0, stream,
                           x + at, RESIDUAL ? residual + at : nullptr, weight, CODES ? static_cast<uint8_t*>(codes) + at : nullptr, CODES ? scales + first * stride_m : nullptr,
                           NORMED ? static_cast<__bf16*>(normed) + at : nullptr, inverse_rms + first, NormShape{here, k, eps, stride_m, stride_k});
        if (const hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

// `partial`: fp32 [parts, k] of scratch, parts = workgroups * rows at a time, both as norm_backward_workgroups and norm_backward_lanes in Python have them.
template <typename G, typename H, typename W, int LANES, int V, bool RESIDUAL, bool WEIGHT>
inline hipError_t launch_rms_norm_backward(const G* grad, const H* h, const W* weight, const float* inverse_rms, const G* grad_residual, G* grad_h, float* partial,
                                           int workgroups, float* grad_weight, bool accumulate, int rows, int k, hipStream_t stream) {
    constexpr int THREADS = LANES > 256 ? LANES : 256, ROWS = THREADS / LANES;
    if (rows < 0 || k <= 0 || k > kNormMostColumns || k % 8 != 0 || k > LANES * V * 8 || workgroups < 1 || workgroups > 1 << 16) return hipErrorInvalidValue;
    if (rows == 0) return hipErrorInvalidValue;
    if (!grad || !h || !weight || !inverse_rms || !grad_h || (RESIDUAL && !grad_residual) || (WEIGHT && (!partial || !grad_weight))) return hipErrorInvalidValue;
    hipLaunchKernelGGL((rms_norm_backward_kernel<G, H, W, LANES, V, RESIDUAL, WEIGHT>), dim3(workgroups), dim3(THREADS), 0, stream, grad, h, weight, inverse_rms,
                       grad_residual, grad_h, partial, rows, k);
    if (const hipError_t rc = hipGetLastError(); rc != hipSuccess || !WEIGHT) return rc;
    hipLaunchKernelGGL(rms_norm_weight_sum_kernel<0>, dim3(ceil_div(k, 32)), dim3(1024), 0, stream, partial, grad_weight, workgroups * ROWS, k, accumulate);
    return hipGetLastError();
}

} // namespace yan
