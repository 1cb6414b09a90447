// Sums and maxima over the lanes that share a token, in registers: a group of 16, 32 or 64 neighbouring lanes of a wave, every one of which
// gets the result. Within a row of 16 by DPP rotations; across rows and halves by the lane swaps of gfx950, which hand both operands of the
// next step to every lane (rows [a b c d] swapped with themselves: [a a c c] and [b b d d]). Every lane of the wave has to be active.
#pragma once

#include "../gemm/utils.hpp"

namespace yan {

constexpr long long kMaxWorkgroups = (1ll << 24) - 1;       // of 256 threads: a launch has less than 2^32 threads

template <int ROTATE>
__device__ __forceinline__ uint32_t rotate_row(uint32_t a) {
    constexpr int ROW_ROR = 0x120;
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(a), ROW_ROR + ROTATE, 0xf, 0xf, true));
}

template <int LANES, typename T, typename Op>
__device__ __forceinline__ T reduce_lanes(T v, Op&& op) {
    static_assert(sizeof(T) == 4 && (LANES == 16 || LANES == 32 || LANES == 64));
    const auto bits = [](T x) { return __builtin_bit_cast(uint32_t, x); };
    const auto value = [](uint32_t x) { return __builtin_bit_cast(T, x); };
    v = op(v, value(rotate_row<8>(bits(v))));
    v = op(v, value(rotate_row<4>(bits(v))));
    v = op(v, value(rotate_row<2>(bits(v))));
    v = op(v, value(rotate_row<1>(bits(v))));
    if constexpr (LANES >= 32) {
        const auto pair = __builtin_amdgcn_permlane16_swap(bits(v), bits(v), false, false);
        v = op(value(pair[0]), value(pair[1]));
    }
    if constexpr (LANES == 64) {
        const auto pair = __builtin_amdgcn_permlane32_swap(bits(v), bits(v), false, false);
        v = op(value(pair[0]), value(pair[1]));
    }
    return v;
}

template <int LANES> __device__ __forceinline__ float sum_lanes(float v) { return reduce_lanes<LANES>(v, [](float a, float b) { return a + b; }); }
template <int LANES> __device__ __forceinline__ int sum_lanes(int v) { return reduce_lanes<LANES>(v, [](int a, int b) { return a + b; }); }
template <int LANES> __device__ __forceinline__ float max_lanes(float v) { return reduce_lanes<LANES>(v, [](float a, float b) { return fmaxf(a, b); }); }
template <int LANES> __device__ __forceinline__ uint32_t max_lanes(uint32_t v) { return reduce_lanes<LANES>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); }

// The maximum over a whole wave as a scalar: rows of 16 as above, then every second row takes its neighbour's, the upper half the lower half's, and the last
// lane has it all (zero, which is what lanes outside of the masks are given, is the least there is). Router, 16384 rows of 256: 16.3 -> 15.8 us.
__device__ __forceinline__ uint32_t max_wave(uint32_t v) {
    constexpr int ROW_BCAST_15 = 0x142, ROW_BCAST_31 = 0x143;
    const auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    v = larger(v, rotate_row<8>(v));
    v = larger(v, rotate_row<4>(v));
    v = larger(v, rotate_row<2>(v));
    v = larger(v, rotate_row<1>(v));
    v = larger(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), ROW_BCAST_15, 0xa, 0xf, false)));
    v = larger(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), ROW_BCAST_31, 0xc, 0xf, false)));
    return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
}

// Across the groups of a wave: every group gets the sum over the lanes that have its place in their groups.
template <int LANES, typename T>
__device__ __forceinline__ T sum_groups(T v) {
    if constexpr (LANES == 16) {
        const auto pair = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
        v = __builtin_bit_cast(T, uint32_t(pair[0])) + __builtin_bit_cast(T, uint32_t(pair[1]));
    }
    if constexpr (LANES <= 32) {
        const auto pair = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
        v = __builtin_bit_cast(T, uint32_t(pair[0])) + __builtin_bit_cast(T, uint32_t(pair[1]));
    }
    return v;
}

} // namespace yan
