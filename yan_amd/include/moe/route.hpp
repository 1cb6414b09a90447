// The router of a mixture-of-experts layer: top-k experts per token with their weights, tokens per expert, balance loss; and its backward.
//
//   l [T, E] logits; s = softmax(l) or sigmoid(l) along a row; the picks of a token are its k largest logits, ties to the lowest expert;
//   w_i = s_i, or s_i / (sum of s over the picks);  c_e = picks of expert e;  n = tokens that are not masked
//   p = s (softmax), s / (sum of s over the row) (sigmoid);  loss = E / (k n^2) sum_e c_e sum_t p[t, e]
//   backward: with g_e = dloss E c_e / (k n^2), c_e taken as a constant, and h_i = dw_i, or (dw_i - sum_j w_j dw_j) / (sum of s over the
//   picks), zero elsewhere:   softmax: dl = s (h + g - sum_e s_e (h_e + g_e));   sigmoid: dl = (1 - s) (s h + p (g - sum_e p_e g_e)),
//   where s h of a renormalised pick is w_i (dw_i - sum_j w_j dw_j)
//
// A group of LANES lanes holds a row, VALUES neighbouring logits a lane, so that lower lanes have lower experts. Picks are made on the logits
// (both scores grow with them) as unsigned keys of the same order: every lane sorts its own, then a round is the maximum over the lanes' first keys, and the
// lowest lane that has it gives up its first. What is summed over tokens, p, stays in the registers of the lane that owns the expert, picks are
// counted in LDS; a workgroup leaves one row of both. Few rows are added up by the workgroup that arrives last, many by a second, small kernel, both in the
// order of the workgroups: no float atomics, the same bits every time.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <algorithm>
#include <limits>
#include <type_traits>

#include "../gemm/scheduler.hpp"
#include "lanes.hpp"

namespace yan {

constexpr int kMaxTopK = 16;            // lane i of a group holds pick i
constexpr int kMaxExperts = 1024;
constexpr int kMaxTokens = 1 << 30;     // so that a launch's last token, rounded up to whole workgroups, is a number of 32 bits

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

// exp(x) for x <= 88, within 2 units in the last place; 0 below -87 (the smallest normal numbers), NaN for NaN. The product with log2(e) is carried to twice
// the bits, its lower part applied to the result: eight instructions, where the library's function cares for every x. A row of 256 logits and 8 picks takes 409 vector
// instructions forward and 266 backward with softmax, 453 and 277 with sigmoid (SQ_INSTS_VALU; 512 logits, sigmoid: 1356 and 365).
__device__ __forceinline__ float exp_of(float x) {
    constexpr float LOG2_E = 1.44269504f, LOG2_E_LOW = 1.92596299e-8f, LN_2 = 0.693147181f;
    const float high = x * LOG2_E, low = fmaf(x, LOG2_E, -high) + x * LOG2_E_LOW;
    const float y = __builtin_amdgcn_exp2f(high);
    return x < -87.f ? 0.f : fmaf(y, low * LN_2, y);
}
// 1 / x for normal numbers, one step of Newton behind the hardware's estimate; and that with 0 for 0
__device__ __forceinline__ float inverse_of_normal(float x) {
    const float r = __builtin_amdgcn_rcpf(x);
    return fmaf(fmaf(-x, r, 1.f), r, r);
}
__device__ __forceinline__ float inverse_of(float x) { return x == 0.f ? 0.f : inverse_of_normal(x); }
constexpr float kMostLogit = std::numeric_limits<float>::max();
__device__ __forceinline__ float finite_top(float top) { return top < -kMostLogit ? 0.f : (top > kMostLogit ? kMostLogit : top); }
// What a row's scores are multiples of. Softmax: exp(top), top the largest logit. Sigmoid: exp(top), top the largest logit where that is below zero, else 1. So the
// largest is not below a half, the sums that scores are divided by are normal numbers, and quotients are as exact in a row of logits all far below zero
// as in any other (from -88 on the scores themselves are less than the smallest normal number, which counts as 0). `unit`, sigmoid: exp(top).
struct ScoreBase {
    float top, unit;
};
template <bool SIGMOID>
__device__ __forceinline__ ScoreBase score_base(float largest) {
    if constexpr (SIGMOID) {
        const float top = fminf(finite_top(largest), 0.f);
        return {top, exp_of(top)};
    }
    return {finite_top(largest), 1.f};
}
// Whether every group of the wave has a lane whose `largest` is zero or more
template <int LANES>
__device__ __forceinline__ bool every_group_reaches_zero(float largest) {
    const unsigned long long have = __ballot(largest >= 0.f);
    if constexpr (LANES == 64) return have != 0;
    const uint32_t low = uint32_t(have), high = uint32_t(have >> 32);
    if constexpr (LANES == 32) return low && high;
    return (low & 0xffff) && low >> 16 && (high & 0xffff) && high >> 16;
}
// A score in multiples of its row's base: sigmoid(l) / unit, or exp(l - top); a logit of +infinity counts as the largest finite number. Sigmoid: `rest` gets 1 - s,
// which near s = 1 is no difference of rounded numbers.
template <bool SIGMOID>
__device__ __forceinline__ float score_of(float l, ScoreBase base, float* rest = nullptr) {
    if constexpr (SIGMOID) {
        // of the magnitude, so that no exponential overflows: 1 / (1 + e^-|l|), or that times e^-|l|, which is t * unit
        const float t = exp_of(fminf(l - base.top, -l)), r = inverse_of_normal(fmaf(t, base.unit, 1.f));
        if (rest) *rest = l < 0.f ? r : t * r;
        return l < 0.f ? t * r : r;
    } else {
        return exp_of((l > kMostLogit ? kMostLogit : l) - base.top);
    }
}

// A row's scores: v are the logits (-infinity past the row's end). Returns their sum, both in multiples of the base (softmax: the sum, by which they have been divided).
// A row of -infinity alone has scores of zero. `rest`: [VALUES], as score_of has it.
template <bool SIGMOID, int LANES, int VALUES>
__device__ __forceinline__ float row_scores(float (&s)[VALUES], const float (&v)[VALUES], ScoreBase base, float* rest = nullptr) {
    float sum = 0.f;
    const auto scores = [&](ScoreBase of) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < VALUES; ++j) {
            s[j] = score_of<SIGMOID>(v[j], of, rest ? rest + j : nullptr);
            sum += s[j];
        }
    };
    // Where all of a wave's rows have a logit of zero or more, as nearly all have, the base is a constant (sigmoid, 16384 rows, backward: 256 logits 12.4 -> 12.2 us, 512
    // 19.4 -> 18.9, 4096 of 1024 18.2 -> 17.3; forward no difference).
    if (SIGMOID && rest && !__any(base.top < 0.f)) scores({0.f, 1.f});
    else scores(base);
    sum = sum_lanes<LANES>(sum);
    if constexpr (!SIGMOID) {
        const float inverse = inverse_of(sum);
#pragma unroll
        for (int j = 0; j < VALUES; ++j) s[j] *= inverse;
    }
    return sum;
}

// The picks of all experts, up to 2^34: sums of the counts' lower 16 bits and of what is above them, neither of which passes 2^26.
struct Picks {
    int low, high;
    __device__ __forceinline__ void add(int count) { low += count & 0xffff, high += count >> 16; }
    template <int LANES>
    __device__ __forceinline__ Picks over_lanes() const { return {sum_lanes<LANES>(low), sum_lanes<LANES>(high)}; }
    __device__ __forceinline__ float number() const { return float((long long)high * 65536 + low); }
};

// What the workgroups of a launch leave for the second kernel: [blocks][E] sums of p, [blocks][E] counts, and per group of 16 experts the
// sums of c p and of c (in two parts); `arrived` counts those groups.
struct RouteWorkspace {
    float* share;
    int* counts;
    float* pull;
    int *picks_low, *picks_high;
    unsigned* arrived;
    __host__ __device__ RouteWorkspace(void* at, int blocks, int e) {
        share = static_cast<float*>(at);
        counts = reinterpret_cast<int*>(share + size_t(blocks) * e);
        pull = reinterpret_cast<float*>(counts + size_t(blocks) * e);
        picks_low = reinterpret_cast<int*>(pull + (e + 15) / 16);
        picks_high = picks_low + (e + 15) / 16;
        arrived = reinterpret_cast<unsigned*>(picks_high + (e + 15) / 16);
    }
    __host__ static size_t bytes(int blocks, int e) { return (size_t(blocks) * e * 2 + 3 * ((e + 15) / 16) + 1) * 4; }
};

__device__ __forceinline__ float balance_loss(float pull, Picks picks, int top_k, int e) {
    const float n = picks.number() / float(top_k);
    return n == 0.f ? 0.f : pull * float(e) / (float(top_k) * n * n);
}

template <typename T, bool SIGMOID, int LANES, int VALUES, int THREADS>
__global__ void __launch_bounds__(THREADS)
moe_route_kernel(const T* __restrict__ logits, const uint8_t* __restrict__ mask, float* __restrict__ weights, int* __restrict__ indices,
                 int* __restrict__ counts, float* __restrict__ loss, void* workspace, int tokens, int e, int top_k, bool renormalize, bool whole, bool join) {
    constexpr int GROUPS = THREADS / LANES, WAVES = THREADS / kWaveSize;
    __shared__ float lds_share[WAVES][LANES * VALUES];
    __shared__ int lds_counts[LANES * VALUES];
    __shared__ uint2 lds_pick[GROUPS][kMaxTopK];
    __shared__ float lds_pull[WAVES];
    __shared__ Picks lds_picks[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, in_group = lane % LANES, first = in_group * VALUES, group_base = lane - in_group;
    float share[VALUES];
#pragma unroll
    for (int j = 0; j < VALUES; ++j) share[j] = 0.f;
    for (int x = threadIdx.x; x < LANES * VALUES; x += THREADS) lds_counts[x] = 0;
    __syncthreads();

    // the logits of a round are loaded in the round before
    float ahead[VALUES];
    const auto load = [&](int t) { load_row(ahead, logits + size_t(t < tokens ? t : 0) * e, first, t < tokens ? e : 0, whole, -std::numeric_limits<float>::infinity()); };
    load(blockIdx.x * GROUPS + int(threadIdx.x) / LANES);
    for (int t0 = blockIdx.x * GROUPS; t0 < tokens; t0 += gridDim.x * GROUPS) {
        const int t = t0 + int(threadIdx.x) / LANES;
        const bool live = t < tokens && (!mask || mask[t]);
        float v[VALUES], s[VALUES];
#pragma unroll
        for (int j = 0; j < VALUES; ++j) v[j] = ahead[j];
        load(t + gridDim.x * GROUPS);
        // this lane's logits in descending order, equal ones in their own; `places`: which they were, four bits each, the first in the lowest
        uint32_t key[VALUES];
        int place[VALUES];
#pragma unroll
        for (int j = 0; j < VALUES; ++j) key[j] = first + j < e ? order_key(v[j]) : 0u, place[j] = j;
#pragma unroll
        for (int round = 0; round < VALUES; ++round)
#pragma unroll
            for (int j = round & 1; j + 1 < VALUES; j += 2) {          // neighbours change places only if the later one is larger: equal ones never do
                const bool swap = key[j + 1] > key[j];
                const uint32_t high = swap ? key[j + 1] : key[j], low = swap ? key[j] : key[j + 1];
                const int p = swap ? place[j + 1] : place[j], q = swap ? place[j] : place[j + 1];
                key[j] = high, key[j + 1] = low, place[j] = p, place[j + 1] = q;
            }
        using Places = std::conditional_t<(VALUES > 8), unsigned long long, uint32_t>;
        Places places = 0;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) places |= Places(place[j]) << (4 * j);
        uint2* const picks = lds_pick[threadIdx.x / LANES];
        float top = 0.f;
#pragma unroll 2
        for (int i = 0; i < top_k; ++i) {
            const uint32_t best = LANES == 64 ? max_wave(key[0]) : max_lanes<LANES>(key[0]);
            const unsigned long long have = __ballot(key[0] == best) >> group_base;
            if (in_group == __ffsll((long long)have) - 1) {
                picks[i] = make_uint2(uint32_t(first) + uint32_t(places & 15), best);
                places >>= 4;
#pragma unroll
                for (int j = 0; j + 1 < VALUES; ++j) key[j] = key[j + 1];
                key[VALUES - 1] = 0u;
            }
            if (i == 0) top = value_of_key(best);
        }
        asm volatile("" ::: "memory");          // a wave's LDS operations are done in order
        const uint2 mine_at = in_group < top_k ? picks[in_group] : make_uint2(0, 0);
        const int my_pick = int(mine_at.x);
        const uint32_t my_key = mine_at.y;
        if (live && in_group < top_k) atomicAdd(&lds_counts[my_pick], 1);
        asm volatile("" ::: "memory");
        const ScoreBase base = score_base<SIGMOID>(top);
        const float sum = row_scores<SIGMOID, LANES>(s, v, base), inverse = inverse_of(sum);
        // lane i has pick i: its score again, from the logit that its key stands for
        float mine = in_group < top_k ? score_of<SIGMOID>(value_of_key(my_key), base) * (SIGMOID ? 1.f : inverse) : 0.f;
        if (renormalize) mine *= inverse_of(sum_lanes<LANES>(mine));
        else if (SIGMOID) mine *= base.unit;
        if (sum != sum) mine = sum;
        if (t < tokens && in_group < top_k) {
            weights[size_t(t) * top_k + in_group] = live ? mine : 0.f;
            indices[size_t(t) * top_k + in_group] = live ? my_pick : -1;
        }
#pragma unroll
        for (int j = 0; j < VALUES; ++j) share[j] += live ? s[j] * (SIGMOID ? inverse : 1.f) : 0.f;
    }

    // the workgroup's row
#pragma unroll
    for (int j = 0; j < VALUES; ++j) {
        share[j] = sum_groups<LANES>(share[j]);
        if (lane < LANES) lds_share[wave][first + j] = share[j];
    }
    __syncthreads();
    const RouteWorkspace to(workspace, gridDim.x, e);
    const bool alone = gridDim.x == 1;
    // Joined here: expert by expert a sum and a count, written and read at device scope, since the workgroups are on different XCDs, whose L2s do not
    // see each other's lines.
    unsigned long long* const meet = reinterpret_cast<unsigned long long*>(static_cast<uint8_t*>(workspace) + kSplitKCounterBytes);
    float pull = 0.f;
    Picks picks{0, 0};
    for (int x = threadIdx.x; x < e; x += THREADS) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += lds_share[w][x];
        const int number = lds_counts[x];
        if (alone) {
            counts[x] = number;
            pull += float(number) * sum;
            picks.add(number);
        } else if (join) {
            __hip_atomic_store(meet + size_t(blockIdx.x) * e + x, uint64_t(uint32_t(number)) << 32 | __builtin_bit_cast(uint32_t, sum), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        } else {
            to.share[size_t(blockIdx.x) * e + x] = sum;
            to.counts[size_t(blockIdx.x) * e + x] = number;
        }
    }
    if (!alone && !join) {
        if (blockIdx.x == 0 && threadIdx.x == 0) *to.arrived = 0;
        return;
    }
    if (!alone) {
        // the workgroup that arrives last adds up, in the order of the workgroups whichever it is, and leaves the counter at zero
        __shared__ unsigned lds_before;
        unsigned* const counter = static_cast<unsigned*>(workspace);
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
        __syncthreads();
        if (threadIdx.x == 0) lds_before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (lds_before != gridDim.x - 1) return;
        if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int x = threadIdx.x; x < e; x += THREADS) {
            float sum = 0.f;
            int number = 0;
            for (int b0 = 0; b0 < int(gridDim.x); b0 += 16) {
                unsigned long long part[16];
#pragma unroll
                for (int b = 0; b < 16; ++b)
                    part[b] = b0 + b < int(gridDim.x) ? __hip_atomic_load(meet + size_t(b0 + b) * e + x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
#pragma unroll
                for (int b = 0; b < 16; ++b) sum += __builtin_bit_cast(float, uint32_t(part[b])), number += int(part[b] >> 32);
            }
            counts[x] = number;
            pull += float(number) * sum;
            picks.add(number);
        }
    }
    pull = sum_lanes<64>(pull), picks = picks.over_lanes<64>();
    if (lane == 0) lds_pull[wave] = pull, lds_picks[wave] = picks;
    __syncthreads();
    if (wave == 0) {
        pull = sum_lanes<16>(lane < WAVES ? lds_pull[lane] : 0.f);
        picks = lane < WAVES ? lds_picks[lane] : Picks{0, 0};
        picks = picks.over_lanes<16>();
        if (lane == 0) *loss = balance_loss(pull, picks, top_k, e);
    }
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
    Picks picks{0, 0};
    picks.add(number);
    picks = picks.over_lanes<16>();
    // Written and read at device scope: the workgroups are on different XCDs, whose L2s do not see each other's lines.
    unsigned before = 0;
    if (threadIdx.x == 0) {
        __hip_atomic_store(from.pull + blockIdx.x, pull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(from.picks_low + blockIdx.x, picks.low, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(from.picks_high + blockIdx.x, picks.high, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
        asm volatile("" ::: "memory");
        before = __hip_atomic_fetch_add(from.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    before = __builtin_amdgcn_readfirstlane(before);
    asm volatile("" ::: "memory");
    if (before != gridDim.x - 1) return;
    pull = 0.f, picks = Picks{0, 0};        // at most kMaxExperts / 16 = 64 groups
    if (threadIdx.x < gridDim.x) {
        pull = __hip_atomic_load(from.pull + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        picks.low = __hip_atomic_load(from.picks_low + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        picks.high = __hip_atomic_load(from.picks_high + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    pull = sum_lanes<64>(pull), picks = picks.over_lanes<64>();
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
        Picks picks{0, 0};
        int c[VALUES];
#pragma unroll
        for (int j = 0; j < VALUES; ++j) c[j] = first + j < e ? counts[first + j] : 0, picks.add(c[j]);
        const float n = picks.template over_lanes<LANES>().number() / float(top_k), scale = grad_loss && n > 0.f ? *grad_loss * float(e) / (float(top_k) * n * n) : 0.f;
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
        // the largest of all lanes is asked for only where it is a base (256 logits 12.2 -> 11.6 us, 512 18.9 -> 18.0)
        ScoreBase base{0.f, 1.f};
        if (!SIGMOID || !every_group_reaches_zero<LANES>(top)) base = score_base<SIGMOID>(max_lanes<LANES>(top));
        float rest[VALUES];
        const float sum = row_scores<SIGMOID, LANES>(s, v, base, rest), inverse = inverse_of(sum);
        // sigmoid: s h, in which the base cancels out where weights are renormalised; softmax: h
        if (renormalize) {
            const float mine = pick < 0 ? 0.f : score_of<SIGMOID>(logit, base) * (SIGMOID ? 1.f : inverse);
            const float part = inverse_of(sum_lanes<LANES>(mine)), weight = mine * part;
            dw = (dw - sum_lanes<LANES>(weight * dw)) * (SIGMOID ? weight : part);
        } else if (SIGMOID) {
            dw *= pick < 0 ? 0.f : score_of<SIGMOID>(logit, base) * base.unit;
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
        const float pull = dot * inverse;           // sigmoid: the sum of p g
#pragma unroll
        for (int j = 0; j < VALUES; ++j) {
            if constexpr (SIGMOID) d[j] = rest[j] * (d[j] + s[j] * ((g[j] - pull) * inverse));
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

// `blocks`: workgroups of the launch. With more than one, `workspace` has RouteWorkspace::bytes(blocks, e) bytes; or, with `join`, it is a split-K workspace
// (kSplitKWorkspaceBytes, its counters at zero), and there is no second kernel.
template <typename T, bool SIGMOID, int LANES, int VALUES, int THREADS>
inline hipError_t launch_moe_route(const T* logits, const uint8_t* mask, float* weights, int* indices, int* counts, float* loss, void* workspace,
                                   int blocks, bool join, int tokens, int e, int top_k, bool renormalize, hipStream_t stream) {
    if (tokens < 0 || tokens > kMaxTokens || e < 1 || e > LANES * VALUES || top_k < 1 || top_k > e || top_k > kMaxTopK || top_k > LANES || blocks < 1) return hipErrorInvalidValue;
    if (!counts || !loss || (tokens && (!logits || !weights || !indices)) || (blocks > 1 && !workspace)) return hipErrorInvalidValue;
    if (join && size_t(blocks) * e * 8 > kSplitKWorkspaceBytes - kSplitKCounterBytes) return hipErrorInvalidValue;
    hipLaunchKernelGGL((moe_route_kernel<T, SIGMOID, LANES, VALUES, THREADS>), dim3(blocks), dim3(THREADS), 0, stream, logits, mask, weights, indices, counts,
                       loss, workspace, tokens, e, top_k, renormalize, rows_in_pieces<VALUES, T>(logits, e), join);
    if (const hipError_t rc = hipGetLastError(); rc != hipSuccess || blocks == 1 || join) return rc;
    hipLaunchKernelGGL(moe_route_finish_kernel<0>, dim3(ceil_div(e, 16)), dim3(1024), 0, stream, counts, loss, workspace, blocks, e, top_k);
    return hipGetLastError();
}

template <typename T, bool SIGMOID, int LANES, int VALUES>
inline hipError_t launch_moe_route_backward(const T* logits, const int* indices, const int* counts, const float* grad_weights, const float* grad_loss,
                                            T* grad_logits, int tokens, int e, int top_k, bool renormalize, hipStream_t stream) {
    if (tokens < 0 || tokens > kMaxTokens || e < 1 || e > LANES * VALUES || top_k < 1 || top_k > kMaxTopK || top_k > LANES) return hipErrorInvalidValue;
    if (tokens == 0) return hipSuccess;
    if (!logits || !indices || !counts || !grad_logits) return hipErrorInvalidValue;
    // as many workgroups as are resident, so that each reads the counts once (fp32, 16384 tokens, 1024 / 2048 / 4096 workgroups: 256 experts 12.1, 11.8, 12.4 us,
    // 512 experts 18.6, 20.8, 25.9; since then 256 take 11.3 with softmax, 11.6 with sigmoid, 512 17.2 and 18.0)
    constexpr int MOST = VALUES > 4 ? 1024 : 2048;
    const int blocks = std::min(ceil_div(tokens, 256 / LANES), MOST);
    hipLaunchKernelGGL((moe_route_backward_kernel<T, SIGMOID, LANES, VALUES>), dim3(blocks), dim3(256), 0, stream, logits, indices,
                       counts, grad_weights, grad_loss, grad_logits, tokens, e, top_k, renormalize,
                       rows_in_pieces<VALUES, T>(logits, e) && rows_in_pieces<VALUES, T>(grad_logits, e));
    return hipGetLastError();
}

} // namespace yan
