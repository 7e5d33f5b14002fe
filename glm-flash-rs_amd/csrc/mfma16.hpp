// The matrix core's 16 x 16 x 32 product of 16-bit operands, and the loads that feed it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.hpp"

namespace gfr {

typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

template <int TYPE>
__device__ __forceinline__ f4_t mfma(uint4 a, uint4 b, f4_t c) {
    if constexpr (TYPE == TYPE_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
}

// Eight values of a row from column k on, zeros from column K on: nothing past K is read, and what lies there (the
// padding of a strided row may hold anything) enters no sum. One 16-byte load at any 2-byte alignment.
__device__ __forceinline__ uint4 load_chunk(const uint16_t* row, int k, int K) {
    uint4 v;
    if (k + 8 <= K) {
        __builtin_memcpy(&v, row + k, 16);
        return v;
    }
    uint32_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = k + j < K ? row[k + j] : 0;
    return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
}

// The same in two steps, for loads that are used later: ask() loads the row's eight values from column k on, or its last
// eight, settle() puts them in place. Only columns from K - 7 on need settle(); K is at least 8 (ask), or anything
// (ask_any, settle_any).
__device__ __forceinline__ uint4 ask(const uint16_t* row, int k, int K) {
    uint4 v;
    __builtin_memcpy(&v, row + min(k, K - 8), 16);
    return v;
}
__device__ __forceinline__ uint4 settle(uint4 v, int k, int K) {
    uint64_t lo = v.x | (uint64_t)v.y << 32, hi = v.z | (uint64_t)v.w << 32;
    const int bits = 16 * (k - min(k, K - 8));
    if (bits >= 64) lo = hi, hi = 0;
    if (bits >= 128) lo = 0;
    if (bits & 63) lo = lo >> (bits & 63) | hi << (64 - (bits & 63)), hi >>= bits & 63;
    return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}
__device__ __forceinline__ uint4 ask_any(const uint16_t* row, int k, int K) {
    return K >= 8 ? ask(row, k, K) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ uint4 settle_any(uint4 v, const uint16_t* row, int k, int K) {
    if (K >= 8) return settle(v, k, K);
    uint64_t lo = 0, hi = 0;
#pragma unroll 1
    for (int j = K - 1; j >= k; --j) hi = hi << 16 | lo >> 48, lo = lo << 16 | row[j];
    return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

}  // namespace gfr
