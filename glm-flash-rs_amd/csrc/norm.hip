// The norms around a block of a layer, with its gate and residual, a row at a time:
//   v = post(x), times gate (or its sigmoid);  h = residual_scale * residual + scale * v;  y = pre(h)
// where a norm is  (z - mean) * 1 / sqrt(mean of squares + eps) * (weight + offset) + bias,  the mean 0 for the RMS kind.
// post, the gate, the residual and pre may each be absent. Statistics and values in fp32, each output rounded once: pre
// takes h as it is before its rounding. Variances are sums of squared differences from the mean, so that they don't cancel.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lanes.hpp"
#include "launch.hpp"
#include "values.hpp"

namespace gfr {
namespace {

// The sum over a row's lanes (L of a wave, or the whole workgroup where L is 0), in all of them. `part`: a buffer that no
// wave may still be reading from the sum before (two in turn are enough: each sum has a barrier).
template <int L>
__device__ __forceinline__ float total(float v, float* part) {
    v = sum_over(L ? L : 64, v);
    if constexpr (L == 0) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = part[0];
        for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v += part[w];
    }
    return v;
}

// V groups of eight columns a lane: group g of lane i starts at column 8 (g lanes + i).
template <int L, int V>
__global__ void __launch_bounds__(L ? 256 : 1024) norm_kernel(NormJob d) {
    __shared__ float part[2][16];
    const int lanes = L ? L : (int)blockDim.x, lane = L ? threadIdx.x % L : threadIdx.x, per = L ? 256 / L : 1;
    int side = 0;
    for (int64_t row = (int64_t)blockIdx.x * per + (L ? threadIdx.x / L : 0); row < d.rows; row += (int64_t)gridDim.x * per) {
        int c[V], count[V];
        Eight ex[V], er[V], eg[V];
        float gate = 1.f;
        if (d.gate && !d.gate_col) gate = load_one(d.gate, d.gate_type, row * d.gate_row);
#pragma unroll
        for (int g = 0; g < V; ++g) {
            c[g] = 8 * (g * lanes + lane), count[g] = d.n - c[g];
            ex[g].a = ex[g].b = er[g].a = er[g].b = eg[g].a = eg[g].b = make_uint4(0, 0, 0, 0);
            if (count[g] > 0) {
                ex[g] = load_some(d.x, d.x_type, row * d.x_stride + c[g], count[g]);
                if (d.residual) er[g] = load_some(d.residual, d.residual_type, row * d.residual_stride + c[g], count[g]);
                if (d.gate && d.gate_col) eg[g] = load_some(d.gate, d.gate_type, row * d.gate_row + c[g], count[g]);
            }
        }
        f8_t v[V];
#pragma unroll
        for (int g = 0; g < V; ++g) v[g] = values(ex[g], d.x_type);
        // v's columns past n are kept at zero up to a norm's weights
        const auto norm = [&](const NormPart& p) {
            Eight ew[V], eb[V];
#pragma unroll
            for (int g = 0; g < V; ++g) {
                ew[g].a = ew[g].b = eb[g].a = eb[g].b = make_uint4(0, 0, 0, 0);
                if (count[g] > 0 && p.weight) ew[g] = load_some(p.weight, p.weight_type, c[g], count[g]);
                if (count[g] > 0 && p.bias) eb[g] = load_some(p.bias, p.bias_type, c[g], count[g]);
            }
            if (p.layer) {
                float s = 0.f;
#pragma unroll
                for (int g = 0; g < V; ++g)
#pragma unroll
                    for (int j = 0; j < 8; ++j) s += v[g][j];
                const float mean = total<L>(s, part[side ^= 1]) * d.per_column;
#pragma unroll
                for (int g = 0; g < V; ++g)
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[g][j] = j < count[g] ? v[g][j] - mean : 0.f;
            }
            float s = 0.f;
#pragma unroll
            for (int g = 0; g < V; ++g)
#pragma unroll
                for (int j = 0; j < 8; ++j) s = fmaf(v[g][j], v[g][j], s);
            const float r = 1.f / sqrtf(total<L>(s, part[side ^= 1]) * d.per_column + p.eps);
#pragma unroll
            for (int g = 0; g < V; ++g) {
                const f8_t w = values(ew[g], p.weight_type), b = values(eb[g], p.bias_type);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[g][j] = p.weight ? v[g][j] * r * (w[j] + p.offset) : v[g][j] * r;
                if (p.bias) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[g][j] += j < count[g] ? b[j] : 0.f;
                }
            }
        };
        if (d.has_post) norm(d.post);
        if (d.gate && !d.gate_col && d.sigmoid) gate = times_logistic(1.f, gate);
#pragma unroll
        for (int g = 0; g < V; ++g) {
            if (d.gate && d.gate_col) {
                const f8_t b = values(eg[g], d.gate_type);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[g][j] *= d.sigmoid ? times_logistic(1.f, b[j]) : b[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[g][j] *= gate;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[g][j] *= d.scale;
            if (d.residual) {
                const f8_t r = values(er[g], d.residual_type);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[g][j] = fmaf(d.residual_scale, r[j], v[g][j]);
            }
            if (d.h && count[g] > 0) store_some(d.h, d.h_type, row * d.h_stride + c[g], v[g], count[g]);
        }
        if (d.y) {
            norm(d.pre);
#pragma unroll
            for (int g = 0; g < V; ++g)
                if (count[g] > 0) store_some(d.y, d.y_type, row * d.y_stride + c[g], v[g], count[g]);
        }
    }
}

template <int L, int V>
hipError_t launch(hipStream_t s, const NormJob& d) {
    const int lanes = (d.n + 8 * V - 1) / (8 * V), threads = L ? 256 : (lanes + 63) / 64 * 64, per = L ? 256 / L : 1;
    const int64_t groups = ((int64_t)d.rows + per - 1) / per;
    norm_kernel<L, V><<<dim3((unsigned)(groups < 1 << 20 ? groups : 1 << 20)), threads, 0, s>>>(d);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_norm(hipStream_t s, NormJob d) {
    d.per_column = 1.f / (float)d.n;
    if (d.n <= 128) return launch<16, 1>(s, d);
    if (d.n <= 512) return launch<64, 1>(s, d);
    if (d.n <= 8192) return launch<0, 1>(s, d);
    if (d.n <= 16384) return launch<0, 2>(s, d);
    return launch<0, 4>(s, d);
}

}  // namespace gfr
