// 16-bit matrix products with their epilogue, for the parts of a model around the EXL3 experts (dense MLP layers, 16-bit
// shared experts, projections):
//   out[r][c] = act(sum over k of x[r][k] w[c][k] + bias[c]) + residual[r][c]
// and the gated form, whose weight holds the gate's rows and then the up matrix's:
//   g = x . w[c] + bias[c], u = x . w[n + c] + bias[n + c]
//   out[r][c] = act(min(g, limit)) * clamp(u, -limit, limit) + residual[r][c]
// x and w in bf16 or fp16; products, sums and the epilogue in fp32, rounded once to out's type.
//
// Weights are the matrix core's A operand and rows its B operand (v_mfma_f32_16x16x32: D holds, in lane l, columns
// 4 (l / 16) .. + 3 of the tile for row l % 16), so that a lane's four results are neighbours in out. A gated tile
// takes 16 gate and 16 up rows in turn, so that a lane holds both halves of its columns.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "launch.hpp"

namespace gfr {
namespace {

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

// ---- epilogue -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float bf16_to_f(uint16_t h) { return __builtin_bit_cast(float, (uint32_t)h << 16); }
__device__ __forceinline__ float f16_to_f(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ __forceinline__ uint16_t f_to_16(float v, int type) {
    return type == TYPE_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ float load_one(const void* p, int type, size_t i) {
    if (type == TYPE_F32) return static_cast<const float*>(p)[i];
    const uint16_t h = static_cast<const uint16_t*>(p)[i];
    return type == TYPE_BF16 ? bf16_to_f(h) : f16_to_f(h);
}
__device__ __forceinline__ f4_t load_four(const void* p, int type, size_t i) {
    if (type == TYPE_F32) return *reinterpret_cast<const f4_t*>(static_cast<const float*>(p) + i);
    const ushort4 h = *reinterpret_cast<const ushort4*>(static_cast<const uint16_t*>(p) + i);
    if (type == TYPE_BF16) return (f4_t){bf16_to_f(h.x), bf16_to_f(h.y), bf16_to_f(h.z), bf16_to_f(h.w)};
    return (f4_t){f16_to_f(h.x), f16_to_f(h.y), f16_to_f(h.z), f16_to_f(h.w)};
}
__device__ __forceinline__ float activate(float v, int act) {
    if (act == ACT_SILU) return v / (1.f + expf(-v));
    if (act == ACT_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    if (act == ACT_GELU_TANH) {
        // 0.5 (1 + tanh(z)) = 1 / (1 + exp(-2 z))
        const float z = 0.79788456080286536f * (v + 0.044715f * v * v * v);
        return v / (1.f + expf(-2.f * z));
    }
    if (act == ACT_RELU) return v < 0.f ? 0.f : v;
    return v;
}
// Four columns c .. c + 3 of row r: those below n are stored. `up` is the gated form's second half.
template <bool GATED>
__device__ __forceinline__ void finish(const DenseJob& d, int r, int c, f4_t v, f4_t up) {
    if (r >= d.rows || c >= d.n) return;
    const bool four = d.vector && c + 3 < d.n;
    f4_t res = {0.f, 0.f, 0.f, 0.f};
    const size_t ra = (size_t)r * d.residual_stride + c, oa = (size_t)r * d.out_stride + c;
    if (d.residual) {
        if (four) {
            res = load_four(d.residual, d.residual_type, ra);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < d.n) res[j] = load_one(d.residual, d.residual_type, ra + j);
        }
    }
    if (d.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < d.n) {
                v[j] += load_one(d.bias, d.bias_type, c + j);
                if constexpr (GATED) up[j] += load_one(d.bias, d.bias_type, (size_t)d.n + c + j);
            }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (GATED) {
            // comparisons that keep a NaN
            const float g = v[j] > d.limit ? d.limit : v[j];
            const float u = up[j] > d.limit ? d.limit : up[j] < -d.limit ? -d.limit : up[j];
            v[j] = activate(g, d.act) * u;
        } else {
            v[j] = activate(v[j], d.act);
        }
        if (d.residual) v[j] += res[j];
    }
    if (d.out_type == TYPE_F32) {
        float* o = static_cast<float*>(d.out) + oa;
        if (four) {
            *reinterpret_cast<f4_t*>(o) = v;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < d.n) o[j] = v[j];
        }
    } else {
        uint16_t* o = static_cast<uint16_t*>(d.out) + oa;
        if (four) {
            *reinterpret_cast<ushort4*>(o) = make_ushort4(f_to_16(v[0], d.out_type), f_to_16(v[1], d.out_type),
                                                          f_to_16(v[2], d.out_type), f_to_16(v[3], d.out_type));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < d.n) o[j] = f_to_16(v[j], d.out_type);
        }
    }
}

// Row of w for row i of a tile whose first output column is c0 (rows past the end: the last one, not stored).
template <bool GATED>
__device__ __forceinline__ int weight_row(const DenseJob& d, int c0, int i) {
    if constexpr (GATED) return min(c0 + (i >> 5) * 16 + (i & 15), d.n - 1) + ((i >> 4) & 1) * d.n;
    return min(c0 + i, d.n - 1);
}

// Eight values of a row from column k on, zeros from column K on: nothing past K is read, and what lies there (the
// padding of a strided row may hold anything) enters no sum. wide: the address is 16-byte aligned at every multiple of 8.
__device__ __forceinline__ uint4 load_chunk(const uint16_t* row, int k, int K, bool wide) {
    if (wide && k + 8 <= K) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = k + j < K ? row[k + j] : 0;
    return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
}

// Any shape, stride and alignment: 64 x 64 tiles, 64 k a step through LDS, four waves of 32 x 32.
template <int TYPE, bool GATED>
__global__ void __launch_bounds__(256) dense_any_kernel(DenseJob d, bool wide) {
    constexpr int LD = 64 + 8;                                     // 16-bit values a tile row in LDS (16 bytes of padding)
    __shared__ __align__(16) uint16_t sw[64 * LD], sx[64 * LD];
    const int tile = blockIdx.x % d.n_tiles;
    const int c0 = tile * (GATED ? 32 : 64), r0 = blockIdx.x / d.n_tiles * 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, a = lane & 15, q = lane >> 4;
    const int wn = (wave & 1) * 32, wr = (wave >> 1) * 32;
    // a thread loads two 8-value chunks of each operand: tile rows i and i + 32, chunk threadIdx.x % 8
    const int i = threadIdx.x >> 3, ch = (threadIdx.x & 7) * 8;
    const uint16_t* wp[2];
    const uint16_t* xp[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        wp[h] = d.w + (size_t)weight_row<GATED>(d, c0, i + 32 * h) * d.w_stride;
        xp[h] = d.x + (size_t)min(r0 + i + 32 * h, d.rows - 1) * d.x_stride;
    }
    f4_t acc[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n) acc[m][n] = (f4_t){0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < d.k; k0 += 64) {
        uint4 vw[2], vx[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            vw[h] = load_chunk(wp[h], k0 + ch, d.k, wide);
            vx[h] = load_chunk(xp[h], k0 + ch, d.k, wide);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            *reinterpret_cast<uint4*>(sw + (i + 32 * h) * LD + ch) = vw[h];
            *reinterpret_cast<uint4*>(sx + (i + 32 * h) * LD + ch) = vx[h];
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint4 fa[2], fb[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                fa[m] = *reinterpret_cast<const uint4*>(sw + (wn + 16 * m + a) * LD + 32 * s + 8 * q);
                fb[m] = *reinterpret_cast<const uint4*>(sx + (wr + 16 * m + a) * LD + 32 * s + 8 * q);
            }
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < 2; ++n) acc[m][n] = mfma<TYPE>(fa[m], fb[n], acc[m][n]);
        }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int r = r0 + wr + 16 * n + a;
        if constexpr (GATED) {
            finish<true>(d, r, c0 + wn / 2 + 4 * q, acc[0][n], acc[1][n]);
        } else {
#pragma unroll
            for (int m = 0; m < 2; ++m) finish<false>(d, r, c0 + wn + 16 * m + 4 * q, acc[m][n], acc[m][n]);
        }
    }
}

bool multiple(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <int TYPE, bool GATED>
hipError_t launch(hipStream_t s, DenseJob d) {
    const bool wide = multiple(d.x, 16) && multiple(d.w, 16) && d.x_stride % 8 == 0 && d.w_stride % 8 == 0;
    constexpr int COLS = GATED ? 32 : 64;
    d.n_tiles = (d.n + COLS - 1) / COLS;
    const int64_t tiles = (int64_t)d.n_tiles * ((d.rows + 63) / 64);
    dense_any_kernel<TYPE, GATED><<<dim3((unsigned)tiles), 256, 0, s>>>(d, wide);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_dense(hipStream_t s, DenseJob d) {
    const auto four = [](const void* p, int type, int64_t stride) {
        return !p || (stride % 4 == 0 && multiple(p, type == TYPE_F32 ? 16 : 8));
    };
    d.vector = four(d.out, d.out_type, d.out_stride) && four(d.residual, d.residual_type, d.residual_stride);
    if (d.type == TYPE_BF16)
        return d.gated ? launch<TYPE_BF16, true>(s, d) : launch<TYPE_BF16, false>(s, d);
    return d.gated ? launch<TYPE_F16, true>(s, d) : launch<TYPE_F16, false>(s, d);
}

}  // namespace gfr
