// Tokens on their way to the experts: every (token, slot) gets a row in the layout that the grouped FP8 GEMMs read, and the token's
// activations go there quantised (1 x 128, the arithmetic and the bits of per_token_cast_kernel).
//
//   rank(t, i) = number of earlier pairs (t', i') that chose the same expert, in the order of t and then i
//   contiguous: row = start_e + rank, where expert e starts at the sum over the experts before it of their counts rounded up to 128
//   masked:     row = e * m_max + rank, for rank < m_max
// Rows past the layout's end (contiguous: M rows, masked: m_max an expert) are not there: such a pair has row -1 and goes nowhere, and so does
// one whose expert is none (below 0 or from E on). Rows that no pair has are left as they were.
//
// Bound by HBM: a token is read once, quantised once and stored top_k times. Few pairs are numbered by every workgroup for itself, one launch;
// many by a histogram of the pairs of each chunk of tokens, a scan along the chunks, and the chunk's own pairs behind that.
#pragma once

#include "../gemm/fp8_cast.hpp"
#include "lanes.hpp"
#include "route.hpp"

namespace yan {

constexpr int kExpertAlignment = 128;
constexpr int kFewPairs = 4096;             // up to here every workgroup counts all pairs itself
constexpr int kTokensPerBlock = 16;         // above: tokens of a chunk
constexpr long long kMaxPairs = (1ll << 31) - (1 << 18);        // so that rows, every expert's rounded up to 128, and a chunk's pairs behind the last token are numbers of 32 bits
static_assert(kMaxPairs + (kExpertAlignment - 1) * kMaxExperts < 1ll << 31 && kMaxPairs + kTokensPerBlock * kMaxTopK < 1ll << 31);
constexpr long long kDispatchCacheBytes = 192ll << 20;

struct DispatchShape {
    int tokens, k_blocks, top_k, experts, m_max;        // m_max 0: contiguous
    int rows;                                           // rows of the layout
    long long stride_g, stride_m, stride_k;             // of the scales, in elements
};

// Starts of the experts' rows out of their counts, in LDS; starts[e] is what they all take. All 256 threads.
__device__ __forceinline__ void align_starts(const int* counts, int* starts, int e) {
    // one wave, 64 experts a step
    if (threadIdx.x < 64) {
        int before = 0;
        for (int x0 = 0; x0 < e; x0 += 64) {
            const int x = x0 + int(threadIdx.x), size = x < e ? ceil_div(counts[x], kExpertAlignment) * kExpertAlignment : 0;
            int sum = size;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int below = __shfl_up(sum, d, 64);
                if (int(threadIdx.x) >= d) sum += below;
            }
            if (x < e) starts[x] = before + sum - size;
            before += __shfl(sum, 63, 64);
        }
        if (threadIdx.x == 0) starts[e] = before;
    }
    __syncthreads();
}

// This workgroup's part of what describes the layout: rows first .. last - 1 of m_indices and, where no pair comes, of `source`.
__device__ __forceinline__ void describe_rows(const int* counts, const int* starts, const DispatchShape& s, int first, int last, int* m_indices, int* source) {
    for (int r = first + int(threadIdx.x); r < last; r += 256) {
        int expert = -1;
        if (r < starts[s.experts]) {
            // the last expert that starts at or before r and has rows: the one before the first that starts behind it
            int low = 0, high = s.experts;
            while (low < high) {
                const int mid = (low + high) / 2;
                if (starts[mid + 1] > r) high = mid; else low = mid + 1;
            }
            expert = low;
        }
        m_indices[r] = expert;
        if (expert < 0 || r - starts[expert] >= counts[expert]) source[r] = -1;
    }
}

// Where a pair's codes and scales start, in bytes and elements; codes below 0: the pair has no row.
struct PairPlace {
    long long codes, scales;
};
__device__ __forceinline__ PairPlace place_of_row(const DispatchShape& s, int row, int expert) {
    const int g = s.m_max ? expert : 0, m = s.m_max ? row - g * s.m_max : row;
    return row < 0 ? PairPlace{-1, 0} : PairPlace{(long long)row * s.k_blocks * 128, g * s.stride_g + m * s.stride_m};
}

// Quantises the blocks of 128 of tokens t0, t0 + 1, ... numbered first .. last - 1 (k_blocks a token) and stores them to their tokens' rows: 16 lanes a
// block, 16 blocks a step, UNROLL steps' loads under way at once. places: [tokens][top_k], of token t0 on. All lanes store a pair's codes, then lane i
// the scale of pair i.
template <int UNROLL, CastStream STREAM, typename T>
__device__ __forceinline__ void scatter_blocks(const T* __restrict__ x, uint8_t* __restrict__ codes, float* __restrict__ scales, const DispatchShape& s, int t0,
                                               int first, int last, const PairPlace* places) {
    const int part = threadIdx.x & 15;
    const T* const from = x + size_t(t0) * s.k_blocks * 128;
    for (int at = first + int(threadIdx.x >> 4); at < last; at += 16 * UNROLL) {
        Raw8<T> raw[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            raw[u] = Raw8<T>{};
            if (at + 16 * u < last) raw[u] = load8<STREAM != kPlain>(from + size_t(at + 16 * u) * 128, part);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int block = at + 16 * u, token = block / s.k_blocks, kb = block - token * s.k_blocks;
            const F32x8 f = to_f32(raw[u]);
            const float amax = fmaxf(max_over_16_lanes(abs_max8(f)), 1e-4f);
            const uint2 q = quantise8(f, kFp8Max / amax);
            if (block >= last) continue;
            const PairPlace* const of = places + token * s.top_k;
            uint8_t* const to = codes + kb * 128;
            for (int i = 0; i < s.top_k; ++i) {
                const long long at_row = of[i].codes;
                if (at_row >= 0) store_codes8<T, STREAM == kStreamBoth>(to + at_row, part, q);
            }
            if (part < s.top_k && of[part].codes >= 0) scales[of[part].scales + kb * s.stride_k] = amax / kFp8Max;
        }
    }
}

__device__ __forceinline__ int row_of_pair(const DispatchShape& s, const int* starts, int expert, int rank) {
    if (s.m_max) return rank < s.m_max ? expert * s.m_max + rank : -1;
    const int row = starts[expert] + rank;
    return row < s.rows ? row : -1;
}

// What the counts say of the layout as a whole: one workgroup's.
__device__ __forceinline__ void describe_experts(const int* counts, const int* starts, const DispatchShape& s, int* offsets, int* masked_m) {
    if (s.m_max) {
        for (int x = threadIdx.x; x < s.experts; x += 256) masked_m[x] = counts[x] < s.m_max ? counts[x] : s.m_max;
    } else {
        for (int x = threadIdx.x; x <= s.experts; x += 256) offsets[x] = starts[x] < s.rows ? starts[x] : s.rows;
    }
}

// Few pairs: `parts` workgroups a token, every one of which goes over all pairs.
template <typename T>
__global__ void __launch_bounds__(256)
moe_dispatch_few_kernel(const T* __restrict__ x, const int* __restrict__ indices, uint8_t* __restrict__ codes, float* __restrict__ scales,
                        int* __restrict__ rows, int* __restrict__ m_indices, int* __restrict__ source, int* __restrict__ offsets, DispatchShape s, int parts) {
    __shared__ int counts[kMaxExperts], before[kMaxExperts], starts[kMaxExperts + 1];
    __shared__ PairPlace places[kMaxTopK];
    const int t = blockIdx.x / parts, piece = blockIdx.x % parts, pairs = s.tokens * s.top_k;
    for (int e = threadIdx.x; e < s.experts; e += 256) counts[e] = before[e] = 0;
    __syncthreads();
    for (int p = threadIdx.x; p < pairs; p += 256) {
        const int e = indices[p];
        if (uint32_t(e) >= uint32_t(s.experts)) continue;
        atomicAdd(&counts[e], 1);
        if (p < t * s.top_k) atomicAdd(&before[e], 1);
    }
    __syncthreads();
    if (!s.m_max) align_starts(counts, starts, s.experts);
    if (int(threadIdx.x) < s.top_k && t < s.tokens) {
        const int* mine = indices + t * s.top_k;
        const int e = mine[threadIdx.x];
        int row = -1;
        if (uint32_t(e) < uint32_t(s.experts)) {
            int rank = before[e];
            for (int i = 0; i < int(threadIdx.x); ++i) rank += mine[i] == e;
            row = row_of_pair(s, starts, e, rank);
        }
        places[threadIdx.x] = place_of_row(s, row, e);
        if (piece == 0) {
            rows[t * s.top_k + threadIdx.x] = row;
            if (!s.m_max && row >= 0) source[row] = t;
        }
    }
    __syncthreads();
    if (!s.m_max) {
        const int share = ceil_div(s.rows, int(gridDim.x)), first = min(s.rows, int(blockIdx.x) * share);
        describe_rows(counts, starts, s, first, min(s.rows, first + share), m_indices, source);
    }
    if (blockIdx.x == 0) describe_experts(counts, starts, s, offsets, m_indices);
    const int share = ceil_div(s.k_blocks, parts);
    if (t < s.tokens) scatter_blocks<2, kPlain>(x, codes, scales, s, t, piece * share, min(s.k_blocks, (piece + 1) * share), places);
}

// Many pairs, first: the histogram of every chunk of tokens, [chunks][E].
template <int = 0>
__global__ void __launch_bounds__(256)
moe_dispatch_count_kernel(const int* __restrict__ indices, int* __restrict__ table, int pairs, int pairs_per_block, int e) {
    __shared__ int counts[kMaxExperts];
    for (int x = threadIdx.x; x < e; x += 256) counts[x] = 0;
    __syncthreads();
    const int first = blockIdx.x * pairs_per_block;
    for (int p = threadIdx.x; p < pairs_per_block && first + p < pairs; p += 256) {
        const int x = indices[first + p];
        if (uint32_t(x) < uint32_t(e)) atomicAdd(&counts[x], 1);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < e; x += 256) table[size_t(blockIdx.x) * e + x] = counts[x];
}

// Second: every entry of the table becomes the sum of those above it, row `blocks` the sum of all. 16 experts a workgroup, 64 threads an expert, each
// with a run of rows, eight of them under way at once; the runs' sums are scanned by a wave an expert.
template <int = 0>
__global__ void __launch_bounds__(1024)
moe_dispatch_scan_kernel(int* __restrict__ table, int blocks, int e) {
    constexpr int TOGETHER = 8;
    __shared__ int sums[64][17];
    const int column = threadIdx.x & 15, part = threadIdx.x >> 4, x = blockIdx.x * 16 + column, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int share = ceil_div(blocks, 64), first = min(blocks, part * share), last = x < e ? min(blocks, first + share) : first;
    const auto load = [&](int (&v)[TOGETHER], int b0) {
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) v[i] = b0 + i < last ? table[size_t(b0 + i) * e + x] : 0;
    };
    int v[TOGETHER], sum = 0;
    for (int b0 = first; b0 < last; b0 += TOGETHER) {
        load(v, b0);
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) sum += v[i];
    }
    sums[part][column] = sum;
    __syncthreads();
    {
        const int mine = sums[lane][wave];
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int below = __shfl_up(upto, d, 64);
            if (lane >= d) upto += below;
        }
        sums[lane][wave] = upto - mine;
    }
    __syncthreads();
    int before = sums[part][column];
    for (int b0 = first; b0 < last; b0 += TOGETHER) {
        if (share > TOGETHER) load(v, b0);          // else they are still here
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) {
            if (b0 + i < last) table[size_t(b0 + i) * e + x] = before;
            before += v[i];
        }
    }
    if (part == 63 && x < e) table[size_t(blocks) * e + x] = before;
}

// Third: the rows of the chunk's pairs and the tokens themselves, by `parts` workgroups a chunk.
template <typename T, CastStream STREAM>
__global__ void __launch_bounds__(256)
moe_dispatch_kernel(const T* __restrict__ x, const int* __restrict__ indices, const int* __restrict__ table, uint8_t* __restrict__ codes,
                    float* __restrict__ scales, int* __restrict__ rows, int* __restrict__ m_indices, int* __restrict__ source, int* __restrict__ offsets,
                    DispatchShape s, int parts) {
    constexpr int PAIRS = kTokensPerBlock * kMaxTopK;
    static_assert(PAIRS == 256, "a thread a pair");
    __shared__ int counts[kMaxExperts], starts[kMaxExperts + 1], expert_of[PAIRS];
    __shared__ PairPlace places[PAIRS];
    // Neighbouring chunks run on one XCD, at about the same time: an expert's scales of one K block are 4 bytes from each of its tokens, and come together to
    // lines in the L2 that way.
    const int chunks = ceil_div(s.tokens, kTokensPerBlock), per_xcd = ceil_div(chunks * parts, kNumXCD);
    const int work = int(blockIdx.x % kNumXCD) * per_xcd + int(blockIdx.x / kNumXCD);
    if (work >= chunks * parts) return;
    const int chunk = work / parts, piece = work - chunk * parts;
    const int t0 = chunk * kTokensPerBlock, here = min(kTokensPerBlock, s.tokens - t0), pairs = here * s.top_k, p = threadIdx.x;
    for (int e = threadIdx.x; e < s.experts; e += 256) counts[e] = table[size_t(chunks) * s.experts + e];
    const int e = p < pairs ? indices[size_t(t0) * s.top_k + p] : -1;
    expert_of[p] = e;
    __syncthreads();
    if (!s.m_max) align_starts(counts, starts, s.experts);
    if (p < pairs) {
        int row = -1;
        if (uint32_t(e) < uint32_t(s.experts)) {
            int rank = table[size_t(chunk) * s.experts + e];
            for (int i = 0; i < p; ++i) rank += expert_of[i] == e;
            row = row_of_pair(s, starts, e, rank);
        }
        places[p] = place_of_row(s, row, e);
        if (piece == 0) {
            rows[size_t(t0) * s.top_k + p] = row;
            if (!s.m_max && row >= 0) source[row] = t0 + p / s.top_k;
        }
    }
    __syncthreads();
    if (!s.m_max) {
        const int share = ceil_div(s.rows, chunks * parts), first = min(s.rows, work * share);
        describe_rows(counts, starts, s, first, min(s.rows, first + share), m_indices, source);
    }
    if (work == 0) describe_experts(counts, starts, s, offsets, m_indices);
    const int blocks = here * s.k_blocks, share = ceil_div(blocks, parts);
    scatter_blocks<4, STREAM>(x, codes, scales, s, t0, piece * share, min(blocks, (piece + 1) * share), places);
}

// Bytes of workspace a launch wants: the table of many pairs.
inline size_t moe_dispatch_workspace_bytes(int tokens, int top_k, int experts) {
    if ((long long)tokens * top_k <= kFewPairs) return 0;
    return (size_t(ceil_div(tokens, kTokensPerBlock)) + 1) * experts * 4;
}

// x [tokens, k] with k = 128 k_blocks; m_max > 0: masked, codes [experts, m_max, k], `m_indices` is masked_m [experts], source and offsets unused;
// m_max == 0: contiguous, codes [rows, k], m_indices and source [rows], offsets [experts + 1].
template <typename T>
inline hipError_t launch_moe_dispatch(const T* x, const int* indices, void* codes, float* scales, long long stride_g, long long stride_m, long long stride_k,
                                      int* rows_of, int* m_indices, int* source, int* offsets, void* workspace, long long workspace_bytes, int tokens, int k,
                                      int top_k, int experts, int m_max, int rows, hipStream_t stream) {
    if (tokens < 0 || k < 128 || k % 128 != 0 || top_k < 1 || top_k > kMaxTopK || experts < 1 || experts > kMaxExperts || m_max < 0 || rows < 0) return hipErrorInvalidValue;
    if (m_max ? rows != experts * m_max : rows % kExpertAlignment != 0) return hipErrorInvalidValue;
    if ((long long)tokens * top_k > kMaxPairs || (long long)experts * m_max >= 1ll << 31) return hipErrorInvalidValue;
    if (m_max ? !m_indices : !offsets) return hipErrorInvalidValue;
    if (tokens && (!x || !indices || !rows_of)) return hipErrorInvalidValue;
    if (rows && (!codes || !scales || (!m_max && (!source || !m_indices)))) return hipErrorInvalidValue;
    const DispatchShape s{tokens, k / 128, top_k, experts, m_max, rows, stride_g, stride_m, stride_k};
    auto* to = static_cast<uint8_t*>(codes);
    const int pairs = tokens * top_k;
    if (pairs <= kFewPairs) {
        // as many workgroups a token as fill the compute units, each with 16 blocks of 128 or more
        const int parts = std::min(ceil_div(k / 128, 16), std::max(1, device_cu_count() / std::max(1, tokens)));
        hipLaunchKernelGGL(moe_dispatch_few_kernel<T>, dim3(std::max(1, tokens) * parts), dim3(256), 0, stream, x, indices, to, scales, rows_of, m_indices, source,
                           offsets, s, parts);
        return hipGetLastError();
    }
    if (!workspace || size_t(workspace_bytes) < moe_dispatch_workspace_bytes(tokens, top_k, experts)) return hipErrorInvalidValue;
    const int blocks = ceil_div(tokens, kTokensPerBlock);
    int* const table = static_cast<int*>(workspace);
    hipLaunchKernelGGL(moe_dispatch_count_kernel<0>, dim3(blocks), dim3(256), 0, stream, indices, table, pairs, kTokensPerBlock * top_k, experts);
    if (const hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
    hipLaunchKernelGGL(moe_dispatch_scan_kernel<0>, dim3(ceil_div(experts, 16)), dim3(1024), 0, stream, table, blocks, experts);
    if (const hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
    // Workgroups a chunk: each has 64 blocks of 128, one step of four loads, or fewer where the chunks are too few for the chip (us with 1, 2, 4, 8, 16:
    // 8192 tokens of 7168 182.5, 175.6, 171.0, 172.5, 166.5; 2048 of 7168 104.7, 66.7, 51.5, 51.6, 47.5; 8192 of 1024 36.7, 31.3, 37.1, 39.4, 46.9; 1024 of 2048
    // 34.1, 23.5, 18.4, 16.6, 16.2)
    const int in_chunk = kTokensPerBlock * s.k_blocks, parts = std::max(ceil_div(in_chunk, 64), std::min(ceil_div(in_chunk, 16), 4 * device_cu_count() / blocks));
    if ((long long)blocks * parts > kMaxWorkgroups - kNumXCD) return hipErrorInvalidValue;
    const int grid = ceil_div(blocks * parts, kNumXCD) * kNumXCD;
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, stream, x, indices, table, to, scales, rows_of, m_indices, source, offsets, s, parts);
        return hipGetLastError();
    };
    if (cast_stream((long long)tokens * k, sizeof(T), true) == kPlain) return launch(moe_dispatch_kernel<T, kPlain>);
    // codes that outgrow the memory-side cache are not found there by the GEMM behind, plain / past the caches (us): 8192 x 8 pairs of 7168, 470 MB, 174.9 / 161.6; 4096 x
    // 8, 224 MB, 93.3 / 84.8, with the product (n 2048) 630 / 627; 8192 x 8 of 2048, 128 MB, 54.0 / 51.7, but with the product (n 1024) 263 / 269
    return (long long)pairs * k > kDispatchCacheBytes ? launch(moe_dispatch_kernel<T, kStreamBoth>) : launch(moe_dispatch_kernel<T, kStreamSource>);
}

} // namespace yan
