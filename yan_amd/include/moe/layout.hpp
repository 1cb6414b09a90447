// The picks of a batch sorted by expert, without padding: what the 16-bit grouped products read (gemm/grouped16.hpp).
//
//   rank(t, i) = number of earlier pairs (t', i') that chose the same expert, in the order of t and then i
//   offsets[e] = pairs of the experts before e;   rows[t, i] = offsets[e] + rank;   source[rows[t, i]] = t
// A pair whose expert is none (below 0 or from E on) has row -1, and `source` is -1 behind the last row.
//
// A thread a pair, 1024 pairs a workgroup. Lanes of a wave with one expert find each other by a ballot a bit of its number; the waves' counts meet in LDS. What
// the pairs in front of the workgroup's add is counted by the workgroup itself for few pairs (one launch), read from a table of the chunks' histograms for more,
// whose columns every workgroup adds up (two), or from that table scanned (three). The experts' starts are scanned by a thread an expert.
// Few bytes: bound by launches, and by the latency of what is in them (256 experts, eight picks: 64 tokens 3.5 us, 1024 5.5, 16384 9.6, 65536 13.9).
#pragma once

#include "dispatch.hpp"

namespace yan {

constexpr int kLayoutChunk = 1024;
constexpr int kLayoutFewChunks = 8;             // up to here every workgroup goes over all pairs itself
constexpr int kLayoutSummedChunks = 256;        // up to here it adds up the table's columns

inline int moe_layout_chunks(long long pairs) { return int(ceil_div<long long>(pairs, kLayoutChunk)); }

// Numbers of 32 bits of workspace a launch wants: those of the largest layouts pass 2 GiB, but not 31 bits.
inline int moe_layout_workspace_numbers(long long pairs, int experts) {
    const int chunks = moe_layout_chunks(pairs);
    return chunks <= kLayoutFewChunks ? 0 : (chunks + 1) * experts;
}
static_assert((kMaxPairs / kLayoutChunk + 2) * kMaxExperts < 1ll << 31);

enum class LayoutCounts { Pairs, Table, ScannedTable };

template <LayoutCounts COUNTS>
__global__ void __launch_bounds__(kLayoutChunk)
moe_layout_kernel(const int* __restrict__ indices, const int* __restrict__ table, int* __restrict__ rows, int* __restrict__ source, int* __restrict__ offsets,
                  int pairs, int top_k, int experts, int chunks) {
    constexpr int WAVES = kLayoutChunk / kWaveSize;
    static_assert(kMaxExperts <= kLayoutChunk);         // a thread an expert
    __shared__ int counts[kMaxExperts], before[kMaxExperts], of_block[WAVES];
    __shared__ uint16_t of_wave[WAVES][kMaxExperts];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, chunk = blockIdx.x;
    const long long first = (long long)chunk * kLayoutChunk;
    const int p = int(min(first + tid, (long long)pairs)), e = p < pairs ? indices[p] : -1;
    const bool real = uint32_t(e) < uint32_t(experts);
    if (tid < experts) counts[tid] = before[tid] = 0;
    for (int x = lane; x < experts; x += kWaveSize) of_wave[wave][x] = 0;
    __syncthreads();
    if constexpr (COUNTS == LayoutCounts::Pairs) {
        for (int q = tid; q < pairs; q += kLayoutChunk) {
            const int x = indices[q];
            if (uint32_t(x) >= uint32_t(experts)) continue;
            atomicAdd(&counts[x], 1);
            if (q < first) atomicAdd(&before[x], 1);
        }
    } else if constexpr (COUNTS == LayoutCounts::Table) {
        // as many threads a column as there are, each with every so many-th row
        const int parts = max(1, kLayoutChunk / experts), part = tid / experts, x = tid - part * experts;
        if (part < parts) {
            int all = 0, above = 0;
#pragma unroll 8
            for (int c = part; c < chunks; c += parts) {
                const int v = table[size_t(c) * experts + x];
                all += v;
                above += c < chunk ? v : 0;
            }
            atomicAdd(&counts[x], all);
            atomicAdd(&before[x], above);
        }
    } else {
        if (tid < experts) {
            counts[tid] = table[size_t(chunks) * experts + tid];
            before[tid] = table[size_t(chunk) * experts + tid];
        }
    }
    // the lanes of this wave with this lane's expert
    unsigned long long same = __ballot(real);
    for (int bit = 0; (experts - 1) >> bit; ++bit) {
        const unsigned long long set = __ballot((e >> bit) & 1);
        same &= (e >> bit) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (real && rank == 0) of_wave[wave][e] = uint16_t(__popcll(same));
    __syncthreads();
    // thread x: pairs of the experts before x, those of its wave's 64 first, and of x itself in the waves in front
    const int size = tid < experts ? counts[tid] : 0;
    int start = size;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int below = __shfl_up(start, d, 64);
        if (lane >= d) start += below;
    }
    if (lane == 63) of_block[wave] = start;
    start -= size;
    if (tid < experts) {
        int in_front = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const int here = of_wave[w][tid];
            of_wave[w][tid] = uint16_t(in_front);
            in_front += here;
        }
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const int here = of_block[w];
        start += w < wave ? here : 0;
        total += here;
    }
    if (tid < experts) before[tid] += start;
    if (chunk == 0) {
        if (tid < experts) offsets[tid] = start;
        if (tid == 0) offsets[experts] = total;
    }
    __syncthreads();
    if (real) {
        const int row = before[e] + of_wave[wave][e] + rank;
        rows[p] = row;
        source[row] = p / top_k;
    } else if (p < pairs) {
        rows[p] = -1;
    }
    if (p < pairs && p >= total) source[p] = -1;
}

// indices [pairs / top_k, top_k], rows likewise, source [pairs], offsets [experts + 1].
inline hipError_t launch_moe_layout(const int* indices, int* rows, int* source, int* offsets, int* workspace, int workspace_numbers, int pairs, int top_k,
                                    int experts, hipStream_t stream) {
    if (pairs < 0 || pairs > kMaxPairs || top_k < 1 || top_k > kMaxTopK || pairs % top_k != 0 || experts < 1 || experts > kMaxExperts || !offsets) return hipErrorInvalidValue;
    if (pairs && (!indices || !rows || !source)) return hipErrorInvalidValue;
    const int chunks = moe_layout_chunks(pairs), grid = std::max(1, chunks);
    int* const table = workspace;
    const auto place = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(kLayoutChunk), 0, stream, indices, table, rows, source, offsets, pairs, top_k, experts, chunks);
        return hipGetLastError();
    };
    if (chunks <= kLayoutFewChunks) return place(moe_layout_kernel<LayoutCounts::Pairs>);
    if (!workspace || workspace_numbers < moe_layout_workspace_numbers(pairs, experts)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(moe_dispatch_count_kernel<0>, dim3(chunks), dim3(256), 0, stream, indices, table, pairs, kLayoutChunk, experts);
    if (const hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
    if (chunks <= kLayoutSummedChunks) return place(moe_layout_kernel<LayoutCounts::Table>);
    hipLaunchKernelGGL(moe_dispatch_scan_kernel<0>, dim3(ceil_div(experts, 16)), dim3(1024), 0, stream, table, chunks, experts);
    if (const hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
    return place(moe_layout_kernel<LayoutCounts::ScannedTable>);
}

} // namespace yan
