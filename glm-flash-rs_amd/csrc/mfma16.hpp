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

// The same in two steps, for loads that are used later, of rows of at least eight values: ask() loads the row's eight values
// from column k on, or its last eight, settle() puts them in place where they are not (columns from K - 7 on).
__device__ __forceinline__ uint4 ask(const uint16_t* row, int k, int K) {
    uint4 v;
    __builtin_memcpy(&v, row + min(k, K - 8), 16);
    return v;
}
// In 32-bit operations: a 64-bit shift that had its amount in the last register of the wave's allocation gave wrong values now
// and then (the compiler may put it there).
__device__ __forceinline__ uint4 settle(uint4 v, int k, int K) {
    const int n = k - min(k, K - 8);                                  // places to move down
    if (n & 4) v.x = v.z, v.y = v.w, v.z = v.w = 0;
    if (n & 2) v.x = v.y, v.y = v.z, v.z = v.w, v.w = 0;
    if (n & 1)
        v = make_uint4(__builtin_amdgcn_alignbit(v.y, v.x, 16), __builtin_amdgcn_alignbit(v.z, v.y, 16),
                       __builtin_amdgcn_alignbit(v.w, v.z, 16), v.w >> 16);
    return n < 8 ? v : make_uint4(0, 0, 0, 0);
}
// Rows of less than eight, a value at a time.
__device__ __forceinline__ uint4 load_short(const uint16_t* row, int k, int K) {
    uint4 v = make_uint4(0, 0, 0, 0);
#pragma unroll 1
    for (int j = K - 1; j >= k; --j)
        v = make_uint4(v.x << 16 | row[j], __builtin_amdgcn_alignbit(v.y, v.x, 16), __builtin_amdgcn_alignbit(v.z, v.y, 16),
                       __builtin_amdgcn_alignbit(v.w, v.z, 16));
    return v;
}

}  // namespace gfr
