// The norms around a block of a layer, with its gate and residual, a row at a time:
//   v = post(x), times gate (or its sigmoid);  h = residual_scale * residual + scale * v;  y = pre(h)
// where a norm is  (z - mean) * 1 / sqrt(mean of squares + eps) * (weight + offset) + bias,  the mean 0 for the RMS kind.
// post, the gate, the residual and pre may each be absent. Statistics and values in fp32, each output rounded once: pre
// takes h as it is before its rounding. Variances are sums of squared differences from the mean, so that they don't cancel.
//
// Bound: HBM, each operand read and each output written once, the row in registers between. 16384 rows of 5120 (bf16 x and
// gate, fp32 stream, both norms) 237 us, 4950 GB/s; 4096 of 4096 (bf16) 23.2, 5790; 65536 of 128 7.1, 4730, of which launch
// and drain are about 3; one of 4096 2.9, two trips to memory. Which lanes hold a row follows its width alone, so that a
// row's results do not depend on the window: 16 lanes up to 128 columns, a wave up to 512, else a workgroup with eight columns
// a lane (with sixteen, half the threads, 16384 x 5120 took 384 us and not 265, one row 4.4 and not 3.4: fewer rows in flight
// for the registers), sixteen over 8192, where eight would need more than 1024 threads, and 32 over 16384, whose operands but x
// are loaded where they are used (registers hold one row). The wide forms have fewer rows under way: the norm alone of 8192 x
// 8200 bf16 88 us, 3040 GB/s, of 8192 x 12288 104, 3870, of 4096 x 16384 65, 4100, of 4096 x 20000 121, 2710, of 4096 x 32768 175,
// 3070; with an fp32 stream 4096 x 16384 156, 5160, 4096 x 32768 354, 4550; 16 rows of 16384 5.1, of 32768 10.7.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lanes.hpp"
#include "launch.hpp"
#include "values.hpp"

// products and sums are rounded as they are written, so that a row has the same bits from either kernel
#pragma clang fp contract(off)

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

// An operand's values where it is either fp32 or of the 16-bit type T (ANY: of any). The branches stay branches: the
// compiler would convert both ways and select, for every operand.
constexpr int ANY = -1;
template <int T>
__device__ __forceinline__ f8_t converted(const Eight& e, int type) {
    if constexpr (T == ANY) return values(e, type);
    f8_t v;
    if (type == TYPE_F32) {
        asm volatile("; fp32");
        v = values(e, TYPE_F32);
    } else {
        asm volatile("; 16 bits");
        v = values(e, T);
    }
    return v;
}
template <int T>
__device__ __forceinline__ void store(void* p, int type, int64_t i, f8_t v, int count) {
    if (T == ANY || type == TYPE_F32) store_some(p, T == ANY ? type : TYPE_F32, i, v, count);
    else store_some(p, T, i, v, count);
}

// V groups of eight columns a lane: group g of lane i starts at column 8 (g lanes + i).
template <int T, int L, int V>
__global__ void __launch_bounds__(L ? 256 : 1024) norm_kernel(NormJob d) {
    constexpr bool LATE = V > 2;                                      // operands at their use: registers hold one row
    __shared__ float part[2][16];
    const int lanes = L ? L : (int)blockDim.x, lane = L ? threadIdx.x % L : threadIdx.x, per = L ? 256 / L : 1;
    const bool ragged = d.n % 8;
    int side = 0;
    // (a loop over rows kept every argument in scalar registers, 62 of which were spilled: 265 us and not 237)
    const int64_t row = d.first + (int64_t)blockIdx.x * per + (L ? threadIdx.x / L : 0);
    if (row >= d.rows) return;
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
            if (!LATE && d.residual) er[g] = load_some(d.residual, d.residual_type, row * d.residual_stride + c[g], count[g]);
            if (!LATE && d.gate && d.gate_col) eg[g] = load_some(d.gate, d.gate_type, row * d.gate_row + c[g], count[g]);
        }
    }
    f8_t v[V];
#pragma unroll
    for (int g = 0; g < V; ++g) v[g] = converted<T>(ex[g], d.x_type);
    // columns past n hold zeros; a norm leaves what it adds to them out again
    const auto clear = [&] {
#pragma unroll
        for (int g = 0; g < V; ++g) {
            if (ragged) {
                asm volatile("; by column");
#pragma unroll
                for (int j = 0; j < 8; ++j) v[g][j] = j < count[g] ? v[g][j] : 0.f;
            } else {
                asm volatile("; by group");
#pragma unroll
                for (int j = 0; j < 8; ++j) v[g][j] = count[g] > 0 ? v[g][j] : 0.f;
            }
        }
    };
    const auto norm = [&](const NormPart& p) {
        Eight ew[V], eb[V];
#pragma unroll
        for (int g = 0; g < V; ++g) {
            ew[g].a = ew[g].b = eb[g].a = eb[g].b = make_uint4(0, 0, 0, 0);
            if (!LATE && count[g] > 0 && p.weight) ew[g] = load_some(p.weight, p.weight_type, c[g], count[g]);
            if (!LATE && count[g] > 0 && p.bias) eb[g] = load_some(p.bias, p.bias_type, c[g], count[g]);
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
                for (int j = 0; j < 8; ++j) v[g][j] -= mean;
            clear();
        }
        float s = 0.f;
#pragma unroll
        for (int g = 0; g < V; ++g)
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fmaf(v[g][j], v[g][j], s);
        const float r = __builtin_amdgcn_rsqf(total<L>(s, part[side ^= 1]) * d.per_column + p.eps);
#pragma unroll
        for (int g = 0; g < V; ++g) {
            if (LATE && count[g] > 0 && p.weight) ew[g] = load_some(p.weight, p.weight_type, c[g], count[g]);
            if (LATE && count[g] > 0 && p.bias) eb[g] = load_some(p.bias, p.bias_type, c[g], count[g]);
            if (p.weight) {
                const f8_t w = converted<T>(ew[g], p.weight_type);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[g][j] = v[g][j] * r * (w[j] + p.offset);
            } else {
                asm volatile("; no weight");
#pragma unroll
                for (int j = 0; j < 8; ++j) v[g][j] *= r;
            }
            if (p.bias) v[g] += converted<T>(eb[g], p.bias_type);  // (zeros past n)
        }
    };
    if (d.has_post) norm(d.post);
    if (d.gate) {
        if (!d.gate_col && d.sigmoid) gate = times_logistic(1.f, gate);
#pragma unroll
        for (int g = 0; g < V; ++g) {
            if (!d.gate_col) {
                asm volatile("; a gate a row");
                v[g] *= gate;
                continue;
            }
            if (LATE && count[g] > 0) eg[g] = load_some(d.gate, d.gate_type, row * d.gate_row + c[g], count[g]);
            f8_t b = converted<T>(eg[g], d.gate_type);
            if (d.sigmoid) {
                asm volatile("; sigmoid");
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = times_logistic(1.f, b[j]);
            }
            v[g] *= b;
        }
    }
    if (d.h || d.residual || d.scale != 1.f) {
#pragma unroll
        for (int g = 0; g < V; ++g) {
            v[g] *= d.scale;
            if (d.residual) {
                if (LATE && count[g] > 0) er[g] = load_some(d.residual, d.residual_type, row * d.residual_stride + c[g], count[g]);
                const f8_t r = converted<T>(er[g], d.residual_type);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[g][j] = fmaf(d.residual_scale, r[j], v[g][j]);
            }
            if (d.h && count[g] > 0) store<T>(d.h, d.h_type, row * d.h_stride + c[g], v[g], count[g]);
        }
    }
    if (d.y) {
        norm(d.pre);
#pragma unroll
        for (int g = 0; g < V; ++g)
            if (count[g] > 0) store<T>(d.y, d.y_type, row * d.y_stride + c[g], v[g], count[g]);
    }
}

// The norm alone, y = pre(x), of many rows: a workgroup keeps the weight and the bias in registers, takes rows in turn and asks
// for the next while it works on one; the kernel above has one load a lane under way and waits for its sums. Columns lie as
// above, and sums are in the same order. (us, above -> here: 16384 x 4096 bf16 60.3 -> 43.6, 6150 GB/s; its layer norm 74.6 ->
// 49; 15935 x 4264 fp16 with an fp32 weight 85 -> 51; 16384 x 8192 165 -> 98; 65536 x 128 8.0 -> 7.1; 1200 x 4096 7.1 -> 6.4. With
// scale, residual and h in it, registers spill: 16384 x 4096 94 -> 102, 5120 with an fp32 stream 182 -> 241.)
template <int T, int L>
__global__ void __launch_bounds__(L ? 256 : 1024, 8) norm_rows_kernel(NormJob d) {
    __shared__ float part[2][16];
    const int lanes = L ? L : (int)blockDim.x, lane = L ? threadIdx.x % L : threadIdx.x, per = L ? 256 / L : 1;
    const NormPart& p = d.pre;
    const int c = 8 * lane, count = d.n - c;
    const int64_t step = (int64_t)gridDim.x * per;
    int side = 0;
    int64_t row = (int64_t)blockIdx.x * per + (L ? threadIdx.x / L : 0);
    if (row >= d.rows) return;
    Eight ex;
    ex.a = ex.b = make_uint4(0, 0, 0, 0);
    const auto ask = [&](int64_t at) {
        if (count > 0) ex = load_some(d.x, d.x_type, at * d.x_stride + c, count);
    };
    ask(row);
    f8_t w = 1.f, b = -0.f;                                           // (-0 leaves a -0 as it is)
    if (count > 0 && p.weight) w = converted<T>(load_some(p.weight, p.weight_type, c, count), p.weight_type) + p.offset;
    if (count > 0 && p.bias) b = converted<T>(load_some(p.bias, p.bias_type, c, count), p.bias_type);
    while (true) {
        f8_t v = converted<T>(ex, d.x_type);
        const int64_t next = row + step < d.rows ? row + step : row;
        ask(next);
        if (p.layer) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
            const float mean = total<L>(s, part[side ^= 1]) * d.per_column;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < count ? v[j] - mean : 0.f;
        }
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(v[j], v[j], s);
        const float root = __builtin_amdgcn_rsqf(total<L>(s, part[side ^= 1]) * d.per_column + p.eps);
        if (count > 0) store<T>(d.y, d.y_type, row * d.y_stride + c, v * root * w + b, count);
        if (next == row) return;
        row = next;
    }
}

// The rows of more threads than the card holds at once; up to what 1024 threads hold at eight columns each.
constexpr int RESIDENT = 256 * 2048;
bool alone(const NormJob& d) {
    return d.n <= 8192 && (int64_t)d.rows * d.n >= (int64_t)8 * RESIDENT && d.y && !d.has_post && !d.gate && !d.residual && !d.h &&
           d.scale == 1.f;
}
template <int T, int L>
hipError_t launch_rows(hipStream_t s, const NormJob& d) {
    const int threads = L ? 256 : (d.n + 511) / 512 * 64, per = L ? 256 / L : 1;
    const int64_t groups = ((int64_t)d.rows + per - 1) / per, most = 256 * (2048 / threads);
    norm_rows_kernel<T, L><<<dim3((unsigned)(groups < most ? groups : most)), threads, 0, s>>>(d);
    return hipGetLastError();
}

template <int T, int L, int V>
hipError_t launch(hipStream_t s, NormJob d) {
    const int lanes = (d.n + 8 * V - 1) / (8 * V), threads = L ? 256 : (lanes + 63) / 64 * 64, per = L ? 256 / L : 1;
    for (; d.first < d.rows; d.first += (int64_t)per << 21) {         // (a launch holds 2^32 threads)
        const int64_t groups = (d.rows - d.first + per - 1) / per;
        norm_kernel<T, L, V><<<dim3((unsigned)(groups < 1 << 21 ? groups : 1 << 21)), threads, 0, s>>>(d);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
template <int T>
hipError_t launch(hipStream_t s, const NormJob& d) {
    if constexpr (T != ANY)
        if (alone(d)) {
            if (d.n <= 128) return launch_rows<T, 16>(s, d);
            return d.n <= 512 ? launch_rows<T, 64>(s, d) : launch_rows<T, 0>(s, d);
        }
    if (d.n <= 128) return launch<T, 16, 1>(s, d);
    if (d.n <= 512) return launch<T, 64, 1>(s, d);
    if (d.n <= 8192) return launch<T, 0, 1>(s, d);
    if (d.n <= 16384) return launch<T, 0, 2>(s, d);
    return launch<T, 0, 4>(s, d);
}

}  // namespace

hipError_t launch_norm(hipStream_t s, NormJob d) {
    d.per_column = 1.f / (float)d.n;
    // the 16-bit type of the operands that are there, if they share one
    const void* const at[] = {d.x, d.residual, d.gate, d.h, d.y, d.post.weight, d.post.bias, d.pre.weight, d.pre.bias};
    const int types[] = {d.x_type, d.residual_type, d.gate_type, d.h_type, d.y_type,
                         d.post.weight_type, d.post.bias_type, d.pre.weight_type, d.pre.bias_type};
    bool bf16 = true, fp16 = true;
    for (int i = 0; i < 9; ++i)
        if (at[i]) bf16 = bf16 && types[i] != TYPE_F16, fp16 = fp16 && types[i] != TYPE_BF16;
    return bf16 ? launch<TYPE_BF16>(s, d) : fp16 ? launch<TYPE_F16>(s, d) : launch<ANY>(s, d);
}

}  // namespace gfr
