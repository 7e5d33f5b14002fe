// Values of 16 and 32 bits in registers, eight neighbours at a time, and the activations of the products' epilogues.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.hpp"

namespace gfr {

// (16: rows in LDS and out are no further aligned)
typedef float f8_t __attribute__((ext_vector_type(8), aligned(16)));
static_assert(alignof(f8_t) == 16, "f8_t's accesses");
__device__ __forceinline__ float bf16_to_f(uint32_t h) { return __builtin_bit_cast(float, h << 16); }
__device__ __forceinline__ float f16_to_f(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }
__device__ __forceinline__ uint32_t f_to_16(float v, int type) {
    return type == TYPE_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ float load_one(const void* p, int type, size_t i) {
    if (type == TYPE_F32) return static_cast<const float*>(p)[i];
    const uint16_t h = static_cast<const uint16_t*>(p)[i];
    return type == TYPE_BF16 ? bf16_to_f(h) : f16_to_f(h);
}
__device__ __forceinline__ void store_one(void* p, int type, size_t i, float v) {
    if (type == TYPE_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = (uint16_t)f_to_16(v, type);
}
// Eight neighbours at an address that is a multiple of 16 bytes, as loaded (the second half: fp32's last four).
struct Eight {
    uint4 a, b;
};
__device__ __forceinline__ Eight load_eight(const void* p, int type, size_t i) {
    Eight e;
    e.a = *reinterpret_cast<const uint4*>(static_cast<const char*>(p) + i * (type == TYPE_F32 ? 4 : 2));
    e.b = make_uint4(0, 0, 0, 0);
    if (type == TYPE_F32) e.b = *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i + 4);
    return e;
}
__device__ __forceinline__ f8_t values(const Eight& e, int type) {
    const uint32_t h[4] = {e.a.x, e.a.y, e.a.z, e.a.w}, g[4] = {e.b.x, e.b.y, e.b.z, e.b.w};
    f8_t v;
    if (type == TYPE_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __builtin_bit_cast(float, h[j]), v[4 + j] = __builtin_bit_cast(float, g[j]);
    } else if (type == TYPE_BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = bf16_to_f(h[j]), v[2 * j + 1] = __builtin_bit_cast(float, h[j] & 0xffff0000u);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = f16_to_f(h[j] & 0xffff), v[2 * j + 1] = f16_to_f(h[j] >> 16);
    }
    return v;
}
__device__ __forceinline__ void store_eight(void* p, int type, size_t i, f8_t v) {
    if (type == TYPE_F32) {
        *reinterpret_cast<f8_t*>(static_cast<float*>(p) + i) = v;
        return;
    }
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = f_to_16(v[2 * j], type) | f_to_16(v[2 * j + 1], type) << 16;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(h[0], h[1], h[2], h[3]);
}
// The same at any address that suits the elements, of the first `count` (from 1 on) of the eight: zeros for the others,
// which are not read.
__device__ __forceinline__ Eight load_some(const void* p, int type, size_t i, int count) {
    const int size = type == TYPE_F32 ? 4 : 2;
    const char* at = static_cast<const char*>(p) + i * size;
    Eight e;
    e.b = make_uint4(0, 0, 0, 0);
    if (count >= 8) {
        __builtin_memcpy(&e.a, at, 16);
        if (type == TYPE_F32) __builtin_memcpy(&e.b, at + 16, 16);
        return e;
    }
    uint32_t w[8];
    if (type == TYPE_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = j < count ? reinterpret_cast<const uint32_t*>(at)[j] : 0;
        e.a = make_uint4(w[0], w[1], w[2], w[3]), e.b = make_uint4(w[4], w[5], w[6], w[7]);
        return e;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = j < count ? reinterpret_cast<const uint16_t*>(at)[j] : 0;
    e.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    return e;
}
__device__ __forceinline__ void store_some(void* p, int type, size_t i, f8_t v, int count) {
    if (count < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) store_one(p, type, i + j, v[j]);
        return;
    }
    char* at = static_cast<char*>(p) + i * (type == TYPE_F32 ? 4 : 2);
    if (type == TYPE_F32) {
        __builtin_memcpy(at, &v, 32);
        return;
    }
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = f_to_16(v[2 * j], type) | f_to_16(v[2 * j + 1], type) << 16;
    __builtin_memcpy(at, h, 16);
}
// v / (1 + exp(-z)) by the hardware's exp2 and reciprocal (one unit each): exp(-z)'s relative error is |z| 2^-23 or so, of
// which the quotient keeps the share exp(-z) / (1 + exp(-z)), so that no value is off by more than 2^-21 of |v|.
__device__ __forceinline__ float times_logistic(float v, float z) {
    return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}
// v times the normal distribution's cumulative function: v h for v < 0 and v (1 - h) else, h = erfc(|v| / sqrt 2) / 2 the tail
// beyond |v|. (0.5 v (1 + erf) cancels below v = -3.) h = exp(-v^2 / 2) t p(t) with t = 1 / (1 + 0.35 |v|): p is a
// polynomial of degree 8 fitted to the scaled complement exp(x^2) erfc(x), within 2^-24.9 of it for |v| to 14, past where h
// is a normal float. The exponential's argument is off by up to 1.5 v^2 2^-24: results below zero by v^2 2^-23 + 2^-20 of
// themselves, others by 2^-20. 4096 x 16384 x 2048 (SiLU 233 us) takes 253 us, 298 with erfcf, 270 with the sum and erff.
__device__ __forceinline__ float gelu(float v) {
    constexpr float P[9] = {0.139621407f, 0.139861867f, 0.119832858f, 0.105508044f, -0.0231099185f,
                            0.159174263f, -0.255714327f, 0.143971726f, -0.0291459356f};
    const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, fabsf(v), 1.f));
    float p = P[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) p = fmaf(p, t, P[i]);
    const float h = p * t * __builtin_amdgcn_exp2f(v * v * -0.72134752044448170f);
    return v * (v < 0.f ? h : 1.f - h);
}
template <int ACT>
__device__ __forceinline__ float activate(float v) {
    if constexpr (ACT == ACT_SILU) return times_logistic(v, v);
    if constexpr (ACT == ACT_GELU) return gelu(v);
    // 0.5 (1 + tanh(z)) = 1 / (1 + exp(-2 z))
    if constexpr (ACT == ACT_GELU_TANH) return times_logistic(v, 1.59576912160573072f * (v + 0.044715f * v * v * v));
    if constexpr (ACT == ACT_RELU) return v < 0.f ? 0.f : v;
    return v;
}
template <int ACT>
__device__ __forceinline__ void activate_eight(f8_t& v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = activate<ACT>(v[j]);
}
// Sums with their bias (and the up matrix's, with its own) to the values before the residual. Comparisons that keep a NaN.
template <bool GATED>
__device__ __forceinline__ f8_t shape(f8_t v, f8_t up, int act, float limit) {
    if constexpr (GATED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = v[j] > limit ? limit : v[j];
            up[j] = up[j] > limit ? limit : up[j] < -limit ? -limit : up[j];
        }
    }
    if (act == ACT_SILU) activate_eight<ACT_SILU>(v);
    else if (act == ACT_GELU) activate_eight<ACT_GELU>(v);
    else if (act == ACT_GELU_TANH) activate_eight<ACT_GELU_TANH>(v);
    else if (act == ACT_RELU) activate_eight<ACT_RELU>(v);
    return GATED ? v * up : v;
}

}  // namespace gfr
