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

#include <stdlib.h>
#include <type_traits>

#include "launch.hpp"
#include "lds_stage.hpp"

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

// Tile of a workgroup. Workgroups go to the 8 XCDs in turn, each with an L2 of its own: an XCD gets a contiguous run of
// tiles, walked in blocks of 4 row tiles through all column tiles, so that the tiles in flight on an XCD share operands.
__device__ __forceinline__ void tile_of(const DenseJob& d, int block, int& tn, int& tr) {
    const int total = gridDim.x, per = total / 8, left = total % 8, x = block % 8;
    const int i = x * per + min(x, left) + block / 8;
    constexpr int G = 4;
    const int r_tiles = total / d.n_tiles, band = i / (G * d.n_tiles), h = min(G, r_tiles - band * G);
    const int j = i - band * G * d.n_tiles;
    tn = j / h;
    tr = band * G + j % h;
}

// ---- tiles through LDS ----------------------------------------------------------------------------------------------
// NT x RT tiles (weight rows x rows), 64 k a step, WN x WR waves of (NT / WN) x (RT / WR). A step's operand rows lie in
// LDS as rows of 128 bytes whose 16-byte chunk c is at position c ^ (row % 8): a direct load's lanes write neighbouring
// positions (lane l: row l / 8, position l % 8), so the lane reads chunk (l % 8) ^ (l / 8) of its row, and the fragment
// reads of 8 neighbouring rows (ds_read_b128) meet 8 different positions, all banks once. LDS holds NSB steps of rows
// and NSA (NSB, or one more) of weights.
// Needs 16-byte aligned rows whose tile lies within 32-bit offsets; k past the last multiple of 64 is staged through
// registers (load_chunk), so that nothing beyond k is read.
template <int NT, int RT, int WN, int WR, int NSA, int NSB>
struct TileShape {
    static constexpr int WAVES = WN * WR, THREADS = 64 * WAVES;
    static constexpr int STAGE_A = NT * 128, STAGE_B = RT * 128, B0 = NSA * STAGE_A;
    static constexpr int MA = NT / WN / 16, NB = RT / WR / 16, LA = NT / 8 / WAVES, LB = RT / 8 / WAVES;
    // the epilogue's transposition: 16 rows of a wave's columns in fp32, padded by 4
    static constexpr int EP_LD = NT / WN + 4, EP_WAVE = 16 * EP_LD * 4;
    static constexpr int STAGES = B0 + NSB * STAGE_B;
    static constexpr int LDS = STAGES > WAVES * EP_WAVE ? STAGES : WAVES * EP_WAVE;
    // this wave's loads that may be in flight when a step's have to have landed
    static constexpr int AHEAD = (NSA - 2) * LA + (NSB - 2) * LB;
    static_assert(NT % (8 * WAVES) == 0 && RT % (8 * WAVES) == 0 && NT % (32 * WN) == 0 && RT % (16 * WR) == 0, "tile");
    static_assert(NSB >= 2 && (NSA == NSB || NSA == NSB + 1) && LDS <= 163840, "stages");
};

template <int TYPE, bool GATED, int NT, int RT, int WN, int WR, int NSA, int NSB>
__global__ void __launch_bounds__(64 * WN * WR) dense_tile_kernel(DenseJob d) {
    using S = TileShape<NT, RT, WN, WR, NSA, NSB>;
    extern __shared__ __align__(1024) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), a = lane & 15, q = lane >> 4;
    int tn, tr;
    tile_of(d, blockIdx.x, tn, tr);
    const int c0 = tn * (GATED ? NT / 2 : NT), r0 = tr * RT;

    // this wave's direct loads, 8 tile rows each: LA of weights, LB of rows
    uint32_t va[S::LA], vb[S::LB];
    const uint32_t chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    const uint64_t wbase = reinterpret_cast<uint64_t>(d.w + (size_t)c0 * d.w_stride);
    const uint64_t ubase = reinterpret_cast<uint64_t>(d.w + (size_t)(d.n + c0) * d.w_stride);
    const uint64_t xbase = reinterpret_cast<uint64_t>(d.x + (size_t)r0 * d.x_stride);
#pragma unroll
    for (int j = 0; j < S::LA; ++j) {
        const int i = (wave * S::LA + j) * 8 + (lane >> 3), c = GATED ? (i >> 5) * 16 + (i & 15) : i;
        va[j] = (uint32_t)min(c, d.n - 1 - c0) * (uint32_t)(d.w_stride * 2) + chunk;
    }
#pragma unroll
    for (int j = 0; j < S::LB; ++j) {
        const int i = (wave * S::LB + j) * 8 + (lane >> 3);
        vb[j] = (uint32_t)min(i, d.rows - 1 - r0) * (uint32_t)(d.x_stride * 2) + chunk;
    }
    const uint32_t lds0 = lds_address(lds);
    // load j of step `step` (a step past the end loads nothing, and counts all the same)
    const int steps = d.k / 64;
    auto issue_a = [&](int j, int step, int stage) {
        const int i = (wave * S::LA + j) * 8;
        const uint64_t base = GATED && (i & 16) ? ubase : wbase;
        load_lds16_s(uniform64(base + (uint64_t)step * 128), va[j],
                     __builtin_amdgcn_readfirstlane(lds0 + stage * S::STAGE_A + i * 128), uniform64(step < steps ? ~0ull : 0ull));
    };
    auto issue_b = [&](int j, int step, int stage) {
        load_lds16_s(uniform64(xbase + (uint64_t)step * 128), vb[j],
                     __builtin_amdgcn_readfirstlane(lds0 + S::B0 + stage * S::STAGE_B + (wave * S::LB + j) * 1024),
                     uniform64(step < steps ? ~0ull : 0ull));
    };

    f4_t acc[S::MA][S::NB];
#pragma unroll
    for (int m = 0; m < S::MA; ++m)
#pragma unroll
        for (int n = 0; n < S::NB; ++n) acc[m][n] = (f4_t){0.f, 0.f, 0.f, 0.f};
    const int wn = wave % WN, wr = wave / WN;
    const char* fa = lds + (wn * (NT / WN) + a) * 128;
    const char* fb = lds + S::B0 + (wr * (RT / WR) + a) * 128;
    auto read_one = [&](int i, int sa, int sb, int s, uint4 (&fra)[S::MA], uint4 (&frb)[S::NB]) {
        const int at = ((4 * s + q) ^ (a & 7)) * 16;
        if (i < S::NB) frb[i] = *reinterpret_cast<const uint4*>(fb + sb * S::STAGE_B + at + i * 2048);
        else fra[i - S::NB] = *reinterpret_cast<const uint4*>(fa + sa * S::STAGE_A + at + (i - S::NB) * 2048);
    };
    // A half step (32 k): its MFMAs on the fragments in hand, and between equal shares of them the reads of the next
    // half's fragments and `loads` direct loads, one by one. In this order and no other: a wave issues in order, so
    // that a burst of loads would hold back its MFMAs until the address units have taken them (16 cycles each, eight
    // waves' worth of them).
    auto half = [&](const uint4 (&ca)[S::MA], const uint4 (&cb)[S::NB], uint4 (&na)[S::MA], uint4 (&nb)[S::NB], int sa, int sb,
                    int s, auto loads, auto&& load) {
        constexpr int READS = S::MA + S::NB, MFMAS = S::MA * S::NB, L = decltype(loads)::value;
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            read_one(i, sa, sb, s, na, nb);
#pragma unroll
            for (int j = (i * L + READS - 1) / READS; j < ((i + 1) * L + READS - 1) / READS; ++j) load(j);
#pragma unroll
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int f = i * MFMAS / READS; f < (i + 1) * MFMAS / READS; ++f)
                acc[f / S::NB][f % S::NB] = mfma<TYPE>(ca[f / S::NB], cb[f % S::NB], acc[f / S::NB][f % S::NB]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // A step's first half loads the weights of step t + NSA - 1 (to the place of step t - 1), its second half the rows of
    // step t + NSB (to its own place). Between the halves every wave's reads of step t are done, and its loads of step
    // t + 1 have landed (loads land in order).
    uint4 a0[S::MA], b0[S::NB], a1[S::MA], b1[S::NB];
#pragma unroll
    for (int p = 0; p < NSB; ++p) {
        if (p < NSA - 1) {
#pragma unroll
            for (int j = 0; j < S::LA; ++j) issue_a(j, p, p);
        }
#pragma unroll
        for (int j = 0; j < S::LB; ++j) issue_b(j, p, p);
    }
    wait_vmcnt<(NSB - 1) * S::LB + (NSA - 2) * S::LA>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < S::MA + S::NB; ++i) read_one(i, 0, 0, 0, a0, b0);
    int sa = 0, sb = 0, last = NSA - 1;
    for (int t = 0; t < steps; ++t) {
        half(a0, b0, a1, b1, sa, sb, 1, std::integral_constant<int, S::LA>{}, [&](int j) { issue_a(j, t + NSA - 1, last); });
        wait_vmcnt<S::AHEAD>();
        lds_barrier();
        const int free_b = sb;
        last = sa;
        sa = sa + 1 == NSA ? 0 : sa + 1;
        sb = sb + 1 == NSB ? 0 : sb + 1;
        // the last step's read of the stage after it is of whatever lies there and is not used
        half(a1, b1, a0, b0, sa, sb, 0, std::integral_constant<int, S::LB>{}, [&](int j) { issue_b(j, t + NSB, free_b); });
    }
    if (d.k % 64) {
        lds_barrier();                                             // the stages are no longer read
        for (int i = threadIdx.x; i < (NT + RT) * 8; i += S::THREADS) {
            const int row = i >> 3, c = i & 7;
            const uint16_t* p = row < NT ? d.w + (size_t)weight_row<GATED>(d, c0, row) * d.w_stride
                                         : d.x + (size_t)min(r0 + row - NT, d.rows - 1) * d.x_stride;
            char* to = row < NT ? lds + sa * S::STAGE_A + row * 128 : lds + S::B0 + sb * S::STAGE_B + (row - NT) * 128;
            *reinterpret_cast<uint4*>(to + (c ^ (row & 7)) * 16) = load_chunk(p, steps * 64 + c * 8, d.k, true);
        }
        lds_barrier();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int i = 0; i < S::MA + S::NB; ++i) read_one(i, sa, sb, s, a0, b0);
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
#pragma unroll
                for (int n = 0; n < S::NB; ++n) acc[m][n] = mfma<TYPE>(a0[m], b0[n], acc[m][n]);
        }
    }

    // Epilogue: a wave's 16 rows at a time through LDS, so that its lanes hold four neighbouring columns of few rows and
    // the residual and out are read and written in whole lines.
    lds_barrier();
    float* ep = reinterpret_cast<float*>(lds + wave * S::EP_WAVE);
    constexpr int COLS = (GATED ? NT / 2 : NT) / WN, QUADS = COLS / 4;
#pragma unroll
    for (int n = 0; n < S::NB; ++n) {
#pragma unroll
        for (int m = 0; m < S::MA; ++m) *reinterpret_cast<f4_t*>(ep + a * S::EP_LD + 16 * m + 4 * q) = acc[m][n];
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int i = lane; i < 16 * QUADS; i += 64) {
            const int row = i / QUADS, c = i % QUADS * 4;
            const float* p = ep + row * S::EP_LD + (GATED ? (c >> 4) * 32 + (c & 15) : c);
            const f4_t v = *reinterpret_cast<const f4_t*>(p);
            const f4_t up = GATED ? *reinterpret_cast<const f4_t*>(p + 16) : v;
            finish<GATED>(d, r0 + wr * (RT / WR) + 16 * n + row, c0 + wn * COLS + c, v, up);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

bool multiple(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <int TYPE, bool GATED, int NT, int RT, int WN, int WR, int NSA, int NSB>
hipError_t launch_tile(hipStream_t s, DenseJob d) {
    using S = TileShape<NT, RT, WN, WR, NSA, NSB>;
    constexpr int COLS = GATED ? NT / 2 : NT;
    d.n_tiles = (d.n + COLS - 1) / COLS;
    const int64_t tiles = (int64_t)d.n_tiles * ((d.rows + RT - 1) / RT);
    dense_tile_kernel<TYPE, GATED, NT, RT, WN, WR, NSA, NSB><<<dim3((unsigned)tiles), S::THREADS, S::LDS, s>>>(d);
    return hipGetLastError();
}

template <int TYPE, bool GATED>
hipError_t launch(hipStream_t s, DenseJob d) {
    const bool wide = multiple(d.x, 16) && multiple(d.w, 16) && d.x_stride % 8 == 0 && d.w_stride % 8 == 0;
    if (wide && d.x_stride < 1 << 22 && d.w_stride < 1 << 22 && d.k >= 64) {
        static const int form = getenv("DENSE_FORM") ? atoi(getenv("DENSE_FORM")) : 0;
        switch (form) {
            case 1: return launch_tile<TYPE, GATED, 256, 256, 4, 2, 2, 2>(s, d);
            case 2: return launch_tile<TYPE, GATED, 256, 256, 4, 2, 3, 2>(s, d);
            case 3: return launch_tile<TYPE, GATED, 128, 128, 2, 2, 2, 2>(s, d);
            case 4: return launch_tile<TYPE, GATED, 128, 128, 2, 4, 4, 4>(s, d);
            case 5: return launch_tile<TYPE, GATED, 256, 128, 4, 2, 3, 3>(s, d);
            case 6: return launch_tile<TYPE, GATED, 128, 256, 2, 4, 3, 3>(s, d);
            case 7: return launch_tile<TYPE, GATED, 128, 128, 2, 4, 3, 2>(s, d);
        }
    }
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
