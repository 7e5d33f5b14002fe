// Sums and maxima over neighbouring lanes of a wave.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "exl3_format.hpp"

namespace gfr {

// ---- reductions over the 2, 4 .. 64 lanes that share a value ---------------------------------------------------------
// Stage by stage each lane meets a lane of the other half of its next larger block (quad swaps, half-row and row
// mirrors, the permlane swaps), so that after the stages up to width w every lane of an aligned block of w has the
// block's result.
template <int STAGE>
__device__ __forceinline__ uint32_t partner(uint32_t v) {
    if constexpr (STAGE == 2) return lane_xor<1>(v);
    else if constexpr (STAGE == 4) return lane_xor<2>(v);
    else if constexpr (STAGE == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, false);   // row_half_mirror
    else if constexpr (STAGE == 16) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, false);  // row_mirror
    else if constexpr (STAGE == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (uint32_t)((__lane_id() & 16) ? r[0] : r[1]);
    } else {
        return lane_xor<32>(v);
    }
}
template <int STAGE, typename T>
__device__ __forceinline__ T partner_of(T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, partner<STAGE>(__builtin_bit_cast(uint32_t, v)));
    } else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, (uint64_t)partner<STAGE>((uint32_t)b) | (uint64_t)partner<STAGE>((uint32_t)(b >> 32)) << 32);
    }
}
template <int STAGE, typename F>
__device__ __forceinline__ void stages_up_to(int width, F f) {
    if constexpr (STAGE <= 64) {
        if (width >= STAGE) f(std::integral_constant<int, STAGE>{});
        stages_up_to<2 * STAGE>(width, f);
    }
}
template <typename T>
__device__ __forceinline__ T larger(T a, T b) { return a > b ? a : b; }
template <typename T>
__device__ __forceinline__ T max_over(int width, T v) {
    stages_up_to<2>(width, [&](auto s) { v = larger(v, partner_of<decltype(s)::value>(v)); });
    return v;
}
template <typename T>
__device__ __forceinline__ T sum_over(int width, T v) {
    stages_up_to<2>(width, [&](auto s) { v += partner_of<decltype(s)::value>(v); });
    return v;
}

// How many lanes before this one have their bit set in a ballot.
__device__ __forceinline__ int set_before(uint64_t ballot) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(ballot >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ballot, 0));
}

}  // namespace gfr
