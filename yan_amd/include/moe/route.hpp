// The router of a mixture-of-experts layer: top-k experts per token with their weights, tokens per expert, balance loss; and its backward.
//
//   l [T, E] logits; s = softmax(l) or sigmoid(l) along a row; the picks of a token are its k largest logits, ties to the lowest expert;
//   w_i = s_i, or s_i / (sum of s over the picks);  c_e = picks of expert e;  n = tokens that are not masked
//   p = s (softmax), s / (sum of s over the row) (sigmoid);  loss = E / (k n^2) sum_e c_e sum_t p[t, e]
//   backward: with g_e = dloss E c_e / (k n^2), c_e taken as a constant, and h_i = dw_i, or (dw_i - sum_j w_j dw_j) / (sum of s over the
//   picks), zero elsewhere:   softmax: dl = s (h + g - sum_e s_e (h_e + g_e));   sigmoid: dl = s (1 - s) (h + (g - sum_e p_e g_e) / sum_e s_e)
//
// A group of LANES lanes holds a row, VALUES neighbouring logits a lane, so that lower lanes have lower experts. Picks are made on the logits
// (both scores grow with them) as unsigned keys of the same order: a round is the maximum over the lane's keys and over the group, and the
// lowest lane that has it takes out its lowest such key and counts it. What is summed over tokens, p and the counts, stays in the registers of the lane
// that owns the expert; a workgroup leaves one row of both, and a second, small kernel adds the rows up in their order: no float atomics, the
// same bits every time.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <limits>

#include "lanes.hpp"

namespace yan {

constexpr int kMaxTopK = 16;            // lane i of a group holds pick i
constexpr int kMaxExperts = 1024;

// The order of floats as the order of unsigned numbers; above 0, which is left for what has been taken out. -0 and 0 are one value. A NaN
// is picked after everything else, as -infinity is (its row's weights are NaN all the same).
__device__ __forceinline__ uint32_t order_key(float x) {
    x = x == x ? x + 0.f : -std::numeric_limits<float>::infinity();
    const int bits = __builtin_bit_cast(int, x);
    return uint32_t(bits) ^ (uint32_t(bits >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of_key(uint32_t key) {
    return __builtin_bit_cast(float, key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__bf16 x) { return float(x); }

// VALUES neighbours of a row from `first` on as fp32, `fill` from element `end` on; by 16 or 8 bytes where `whole` says that rows allow it
template <int VALUES, typename T>
__device__ __forceinline__ void load_row(float (&v)[VALUES], const T* row, int first, int end, bool whole, float fill) {
    constexpr int PIECE = VALUES * sizeof(T) >= 16 ? 16 / sizeof(T) : VALUES;         // elements an instruction takes
    typedef T Vec __attribute__((ext_vector_type(PIECE == 1 ? 2 : PIECE)));
    if (PIECE > 1 && whole) {
#pragma unroll
        for (int p = 0; p < VALUES; p += PIECE) {
            Vec piece{};
            const bool live = first + p < end;
            if (live) piece = *reinterpret_cast<const Vec*>(row + first + p);
#pragma unroll
            for (int j = 0; j < PIECE; ++j) v[p + j] = live ? to_float(piece[j]) : fill;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < VALUES; ++j) v[j] = first + j < end ? to_float(row[first + j]) : fill;
}
// whether load_row may take whole pieces: pieces do not cross the end of a row and start at multiples of their size
template <int VALUES, typename T>
__host__ __device__ inline bool rows_in_pieces(const void* base, int e) {
    constexpr int PIECE = VALUES * sizeof(T) >= 16 ? 16 / sizeof(T) : VALUES;
    return e % PIECE == 0 && reinterpret_cast<uintptr_t>(base) % (PIECE * sizeof(T)) == 0;
}

// A row's scores: v are the logits (-infinity past the row's end), `top` the largest; returns their sum. A logit of +infinity counts as the
// largest finite number; a row of -infinity alone has scores of zero.
template <bool SIGMOID, int LANES, int VALUES>
__device__ __forceinline__ float row_scores(float (&s)[VALUES], const float (&v)[VALUES], float top) {
    constexpr float MOST = std::numeric_limits<float>::max();
    top = top < -MOST ? 0.f : (top > MOST ? MOST : top);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < VALUES; ++j) {
        const float l = v[j] > MOST ? MOST : v[j];
        s[j] = SIGMOID ? 1.f / (1.f + expf(-l)) : expf(l - top);
        sum += s[j];
    }
    sum = sum_lanes<LANES>(sum);
    if constexpr (!SIGMOID) {
        const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) s[j] *= inverse;
    }
    return sum;
}

// What the workgroups of a launch leave for the second kernel: [blocks][E] sums of p, [blocks][E] counts, and per group of 16 experts the
// sums of c p and of c; `arrived` counts those groups.
struct RouteWorkspace {
    float* share;
    int* counts;
    float* pull;
    int* picks;
    unsigned* arrived;
    __host__ __device__ RouteWorkspace(void* at, int blocks, int e) {
        share = static_cast<float*>(at);
        counts = reinterpret_cast<int*>(share + size_t(blocks) * e);
        pull = reinterpret_cast<float*>(counts + size_t(blocks) * e);
        picks = reinterpret_cast<int*>(pull + (e + 15) / 16);
        arrived = reinterpret_cast<unsigned*>(picks + (e + 15) / 16);
    }
    __host__ static size_t bytes(int blocks, int e) { return (size_t(blocks) * e * 2 + 2 * ((e + 15) / 16) + 1) * 4; }
};

__device__ __forceinline__ float balance_loss(float pull, int picks, int top_k, int e) {
    const float n = float(picks) / float(top_k);
    return picks == 0 ? 0.f : pull * float(e) / (float(top_k) * n * n);
}

template <typename T, bool SIGMOID, int LANES, int VALUES>
__global__ void __launch_bounds__(256)
moe_route_kernel(const T* __restrict__ logits, const uint8_t* __restrict__ mask, float* __restrict__ weights, int* __restrict__ indices,
                 int* __restrict__ counts, float* __restrict__ loss, void* workspace, int tokens, int e, int top_k, bool renormalize, bool whole) {
    constexpr int GROUPS = 256 / LANES;
    __shared__ float lds_share[4][LANES * VALUES];
    __shared__ int lds_counts[4][LANES * VALUES];
    __shared__ float lds_pull[4];
    __shared__ int lds_picks[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, in_group = lane % LANES, first = in_group * VALUES, group_base = lane - in_group;
    float share[VALUES];
    int count[VALUES];
#pragma unroll
    for (int j = 0; j < VALUES; ++j) share[j] = 0.f, count[j] = 0;

    for (int t0 = blockIdx.x * GROUPS; t0 < tokens; t0 += gridDim.x * GROUPS) {
        const int t = t0 + int(threadIdx.x) / LANES;
        const bool live = t < tokens && (!mask || mask[t]);
        float v[VALUES], s[VALUES];
        load_row(v, logits + size_t(t < tokens ? t : 0) * e, first, e, whole, -std::numeric_limits<float>::infinity());
        uint32_t key[VALUES];
#pragma unroll
        for (int j = 0; j < VALUES; ++j) key[j] = first + j < e ? order_key(v[j]) : 0u;
        uint32_t my_key = 0;
        int my_pick = 0;
        float top = 0.f;
        for (int i = 0; i < top_k; ++i) {
            uint32_t mine = key[0];
#pragma unroll
            for (int j = 1; j < VALUES; ++j) mine = mine > key[j] ? mine : key[j];
            const uint32_t best = max_lanes<LANES>(mine);
            const unsigned long long have = __ballot(mine == best) >> group_base;
            const int winner = __ffsll((long long)have) - 1;
            int place = 0;
            bool open = in_group == winner;
#pragma unroll
            for (int j = 0; j < VALUES; ++j) {
                const bool hit = open && key[j] == best;
                place = hit ? j : place;
                key[j] = hit ? 0u : key[j];
                count[j] += hit && live;
                open = open && !hit;
            }
            const int pick = __shfl(first + place, group_base + winner, 64);
            if (i == 0) top = value_of_key(best);
            if (in_group == i) my_key = best, my_pick = pick;
        }
        const float sum = row_scores<SIGMOID, LANES>(s, v, top);
        // lane i has pick i: its score again, from the logit that its key stands for
        float mine = 0.f;
        {
            constexpr float MOST = std::numeric_limits<float>::max();
            const float t_ = top < -MOST ? 0.f : (top > MOST ? MOST : top), l = fminf(value_of_key(my_key), MOST);
            if (in_group < top_k) mine = SIGMOID ? 1.f / (1.f + expf(-l)) : expf(l - t_) * (sum == 0.f ? 0.f : 1.f / sum);
            if (sum != sum) mine = sum;
        }
        if (renormalize) {
            const float chosen = sum_lanes<LANES>(in_group < top_k ? mine : 0.f);
            mine = chosen == 0.f ? 0.f : mine / chosen;
        }
        if (t < tokens && in_group < top_k) {
            weights[size_t(t) * top_k + in_group] = live ? mine : 0.f;
            indices[size_t(t) * top_k + in_group] = live ? my_pick : -1;
        }
        const float part = !live ? 0.f : SIGMOID ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) share[j] += live ? s[j] * part : 0.f;
    }

    // the workgroup's row
#pragma unroll
    for (int j = 0; j < VALUES; ++j) {
        share[j] = sum_groups<LANES>(share[j]);
        count[j] = sum_groups<LANES>(count[j]);
        if (lane < LANES) lds_share[wave][first + j] = share[j], lds_counts[wave][first + j] = count[j];
    }
    __syncthreads();
    const RouteWorkspace to(workspace, gridDim.x, e);
    const bool alone = gridDim.x == 1;
    float pull = 0.f;
    int picks = 0;
    for (int x = threadIdx.x; x < e; x += 256) {
        const float sum = (lds_share[0][x] + lds_share[1][x]) + (lds_share[2][x] + lds_share[3][x]);
        const int number = lds_counts[0][x] + lds_counts[1][x] + lds_counts[2][x] + lds_counts[3][x];
        if (alone) {
            counts[x] = number;
            pull += float(number) * sum;
            picks += number;
        } else {
            to.share[size_t(blockIdx.x) * e + x] = sum;
            to.counts[size_t(blockIdx.x) * e + x] = number;
        }
    }
    if (!alone) {
        if (blockIdx.x == 0 && threadIdx.x == 0) *to.arrived = 0;
        return;
    }
    pull = sum_lanes<64>(pull), picks = sum_lanes<64>(picks);
    if (lane == 0) lds_pull[wave] = pull, lds_picks[wave] = picks;
    __syncthreads();
    if (threadIdx.x == 0)
        *loss = balance_loss((lds_pull[0] + lds_pull[1]) + (lds_pull[2] + lds_pull[3]), lds_picks[0] + lds_picks[1] + lds_picks[2] + lds_picks[3], top_k, e);
}

// Adds up the workgroups' rows, 16 experts a workgroup; the last workgroup to arrive adds up what the loss takes of each, in their order.
template <int = 0>
__global__ void __launch_bounds__(1024)
moe_route_finish_kernel(int* __restrict__ counts, float* __restrict__ loss, void* workspace, int blocks, int e, int top_k) {
    __shared__ float lds_share[64][16];
    __shared__ int lds_counts[64][16];
    const RouteWorkspace from(workspace, blocks, e);
    const int column = threadIdx.x & 15, part = threadIdx.x >> 4, x = blockIdx.x * 16 + column;
    float share = 0.f;
    int number = 0;
    if (x < e)
        for (int b = part; b < blocks; b += 64) share += from.share[size_t(b) * e + x], number += from.counts[size_t(b) * e + x];
    lds_share[part][column] = share, lds_counts[part][column] = number;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    // one wave: lane 16 q + c adds up the parts 16 q .. 16 q + 15 of column c
    share = 0.f, number = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) share += lds_share[(part & 3) * 16 + i][column], number += lds_counts[(part & 3) * 16 + i][column];
    share = sum_groups<16>(share), number = sum_groups<16>(number);
    if (threadIdx.x < 16 && x < e) counts[x] = number;
    float pull = sum_lanes<16>(float(number) * share);
    int picks = sum_lanes<16>(number);
    // Written and read at device scope: the workgroups are on different XCDs, whose L2s do not see each other's lines.
    unsigned before = 0;
    if (threadIdx.x == 0) {
        __hip_atomic_store(from.pull + blockIdx.x, pull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(from.picks + blockIdx.x, picks, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
        asm volatile("" ::: "memory");
        before = __hip_atomic_fetch_add(from.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    before = __builtin_amdgcn_readfirstlane(before);
    asm volatile("" ::: "memory");
    if (before != gridDim.x - 1) return;
    pull = 0.f, picks = 0;                  // at most kMaxExperts / 16 = 64 groups
    if (threadIdx.x < gridDim.x) {
        pull = __hip_atomic_load(from.pull + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        picks = __hip_atomic_load(from.picks + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    pull = sum_lanes<64>(pull), picks = sum_lanes<64>(picks);
    if (threadIdx.x == 0) *loss = balance_loss(pull, picks, top_k, e);
}

template <typename T, bool SIGMOID, int LANES, int VALUES>
__global__ void __launch_bounds__(256)
moe_route_backward_kernel(const T* __restrict__ logits, const int* __restrict__ indices, const int* __restrict__ counts,
                          const float* __restrict__ grad_weights, const float* __restrict__ grad_loss, T* __restrict__ grad_logits, int tokens, int e,
                          int top_k, bool renormalize, bool whole) {
    constexpr int GROUPS = 256 / LANES;
    __shared__ float lds_h[GROUPS][LANES * VALUES];
    const int lane = threadIdx.x & 63, in_group = lane % LANES, first = in_group * VALUES;
    float* const h_row = lds_h[threadIdx.x / LANES];

    // g: the balance loss's pull on the share of each of this lane's experts
    float g[VALUES];
    {
        int picks = 0, c[VALUES];
#pragma unroll
        for (int j = 0; j < VALUES; ++j) c[j] = first + j < e ? counts[first + j] : 0, picks += c[j];
        picks = sum_lanes<LANES>(picks);
        const float n = float(picks) / float(top_k), scale = grad_loss && picks ? *grad_loss * float(e) / (float(top_k) * n * n) : 0.f;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) g[j] = scale * float(c[j]);
    }
    for (int t0 = blockIdx.x * GROUPS; t0 < tokens; t0 += gridDim.x * GROUPS) {
        const int t = t0 + int(threadIdx.x) / LANES;
        const size_t row = size_t(t < tokens ? t : 0);
        float v[VALUES], s[VALUES];
        load_row(v, logits + row * e, first, e, whole, -std::numeric_limits<float>::infinity());
        // lane i: pick i, its logit and the gradient of its weight. A token without a first pick is a masked one.
        int pick = -1;
        float dw = 0.f, logit = -std::numeric_limits<float>::infinity();
        if (in_group < top_k) {
            pick = indices[row * top_k + in_group];
            if (uint32_t(pick) >= uint32_t(e)) pick = -1;
            if (pick >= 0) {
                logit = to_float(logits[row * e + pick]);
                if (grad_weights) dw = grad_weights[row * top_k + in_group];
            }
        }
        const bool live = __shfl(pick, lane - in_group, 64) >= 0;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) h_row[first + j] = 0.f;
        float top = v[0];
#pragma unroll
        for (int j = 1; j < VALUES; ++j) top = fmaxf(top, v[j]);
        top = max_lanes<LANES>(top);
        const float sum = row_scores<SIGMOID, LANES>(s, v, top);
        if (renormalize) {
            constexpr float MOST = std::numeric_limits<float>::max();
            const float t_ = top < -MOST ? 0.f : (top > MOST ? MOST : top), l = fminf(logit, MOST);
            float mine = SIGMOID ? 1.f / (1.f + expf(-l)) : expf(l - t_) * (sum == 0.f ? 0.f : 1.f / sum);
            if (pick < 0) mine = 0.f;
            const float chosen = sum_lanes<LANES>(mine), inverse = chosen == 0.f ? 0.f : 1.f / chosen;
            dw = (dw - sum_lanes<LANES>(mine * inverse * dw)) * inverse;
        }
        asm volatile("" ::: "memory");              // a wave's LDS operations are done in order: the zeros, the picks, then the reads
        if (pick >= 0) h_row[pick] = dw;
        asm volatile("" ::: "memory");
        float d[VALUES], dot = 0.f;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) {
            d[j] = h_row[first + j] + (SIGMOID ? 0.f : g[j]);
            dot += s[j] * (SIGMOID ? g[j] : d[j]);
        }
        asm volatile("" ::: "memory");
        dot = sum_lanes<LANES>(dot);
        const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) {
            if constexpr (SIGMOID) d[j] = s[j] * (1.f - s[j]) * (d[j] + (g[j] - dot * inverse) * inverse);
            else d[j] = s[j] * (d[j] - dot);
            if (!live) d[j] = 0.f;
        }
        if (t >= tokens) continue;
        constexpr int PIECE = VALUES * sizeof(T) >= 16 ? 16 / sizeof(T) : VALUES;
        typedef T Vec __attribute__((ext_vector_type(PIECE == 1 ? 2 : PIECE)));
        T* const out = grad_logits + row * e;
        if (PIECE > 1 && whole) {
#pragma unroll
            for (int p = 0; p < VALUES; p += PIECE) {
                Vec piece;
#pragma unroll
                for (int j = 0; j < PIECE; ++j) piece[j] = static_cast<T>(d[p + j]);
                if (first + p < e) *reinterpret_cast<Vec*>(out + first + p) = piece;
            }
        } else {
#pragma unroll
            for (int j = 0; j < VALUES; ++j)
                if (first + j < e) out[first + j] = static_cast<T>(d[j]);
        }
    }
}

// `blocks`: workgroups of the launch; with more than one, `workspace` has RouteWorkspace::bytes(blocks, e) bytes.
template <typename T, bool SIGMOID, int LANES, int VALUES>
inline hipError_t launch_moe_route(const T* logits, const uint8_t* mask, float* weights, int* indices, int* counts, float* loss, void* workspace,
                                   int blocks, int tokens, int e, int top_k, bool renormalize, hipStream_t stream) {
    if (tokens < 0 || e < 1 || e > LANES * VALUES || top_k < 1 || top_k > e || top_k > kMaxTopK || top_k > LANES || blocks < 1) return hipErrorInvalidValue;
    if (!logits || !weights || !indices || !counts || !loss || (blocks > 1 && !workspace)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((moe_route_kernel<T, SIGMOID, LANES, VALUES>), dim3(blocks), dim3(256), 0, stream, logits, mask, weights, indices, counts, loss,
                       workspace, tokens, e, top_k, renormalize, rows_in_pieces<VALUES, T>(logits, e));
    if (const hipError_t rc = hipGetLastError(); rc != hipSuccess || blocks == 1) return rc;
    hipLaunchKernelGGL(moe_route_finish_kernel<0>, dim3(ceil_div(e, 16)), dim3(1024), 0, stream, counts, loss, workspace, blocks, e, top_k);
    return hipGetLastError();
}

template <typename T, bool SIGMOID, int LANES, int VALUES>
inline hipError_t launch_moe_route_backward(const T* logits, const int* indices, const int* counts, const float* grad_weights, const float* grad_loss,
                                            T* grad_logits, int tokens, int e, int top_k, bool renormalize, hipStream_t stream) {
    if (tokens < 0 || e < 1 || e > LANES * VALUES || top_k < 1 || top_k > kMaxTopK || top_k > LANES) return hipErrorInvalidValue;
    if (tokens == 0) return hipSuccess;
    if (!logits || !indices || !counts || !grad_logits) return hipErrorInvalidValue;
    const int blocks = ceil_div(tokens, 256 / LANES);
    hipLaunchKernelGGL((moe_route_backward_kernel<T, SIGMOID, LANES, VALUES>), dim3(blocks < 2048 ? blocks : 2048), dim3(256), 0, stream, logits, indices,
                       counts, grad_weights, grad_loss, grad_logits, tokens, e, top_k, renormalize,
                       rows_in_pieces<VALUES, T>(logits, e) && rows_in_pieces<VALUES, T>(grad_logits, e));
    return hipGetLastError();
}

} // namespace yan
