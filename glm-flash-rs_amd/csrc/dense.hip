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
#include "lds_stage.hpp"
#include "mfma16.hpp"
#include "values.hpp"

namespace gfr {
namespace {

// ---- epilogue -------------------------------------------------------------------------------------------------------
// Up to COUNT (4 or 8) columns c .. of row r, element by element: any alignment, and the last columns. Where the tensors
// allow it, four columns take one load and one store.
template <bool GATED, int COUNT>
__device__ __forceinline__ void finish_some(const DenseJob& d, int r, int c, f8_t v, f8_t up) {
    const size_t ra = (size_t)r * d.residual_stride + c, oa = (size_t)r * d.out_stride + c;
    const int count = min(COUNT, d.n - c);
    if (d.bias) {
#pragma unroll
        for (int j = 0; j < COUNT; ++j)
            if (j < count) {
                v[j] += load_one(d.bias, d.bias_type, c + j);
                if constexpr (GATED) up[j] += load_one(d.bias, d.bias_type, (size_t)d.n + c + j);
            }
    }
    v = shape<GATED>(v, up, d.act, d.limit);
    if (COUNT == 4 && d.vector && count == 4) {
        if (d.residual) {
            const float4 f = d.residual_type == TYPE_F32 ? *reinterpret_cast<const float4*>(static_cast<const float*>(d.residual) + ra)
                                                         : make_float4(0.f, 0.f, 0.f, 0.f);
            v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
            if (d.residual_type != TYPE_F32) {
                const ushort4 h = *reinterpret_cast<const ushort4*>(static_cast<const uint16_t*>(d.residual) + ra);
                const bool bf = d.residual_type == TYPE_BF16;
                v[0] += bf ? bf16_to_f(h.x) : f16_to_f(h.x), v[1] += bf ? bf16_to_f(h.y) : f16_to_f(h.y);
                v[2] += bf ? bf16_to_f(h.z) : f16_to_f(h.z), v[3] += bf ? bf16_to_f(h.w) : f16_to_f(h.w);
            }
        }
        if (d.out_type == TYPE_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(d.out) + oa) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(d.out) + oa) =
                make_uint2(f_to_16(v[0], d.out_type) | f_to_16(v[1], d.out_type) << 16,
                           f_to_16(v[2], d.out_type) | f_to_16(v[3], d.out_type) << 16);
        return;
    }
#pragma unroll
    for (int j = 0; j < COUNT; ++j)
        if (j < count) {
            if (d.residual) v[j] += load_one(d.residual, d.residual_type, ra + j);
            store_one(d.out, d.out_type, oa + j, v[j]);
        }
}

// The epilogue of a wave's RB x COLS results (COLS columns from c0 on, rows from r0 on), which lie in LDS as RB rows of LD
// floats (a gated tile's 16 gate and 16 up columns in turn): eight columns a lane, so that the residual and out are read
// and written in whole lines. Plain sums: all passes' residuals in flight at once; else one pass ahead, in a loop (the
// activations' code once: unrolled it spilled the sums).
template <bool GATED, int COLS, int RB, int LD>
__device__ __forceinline__ void finish_rows(const DenseJob& d, const float* ep, int r0, int c0) {
    constexpr int LANES = COLS / 8, ROWS = 64 / LANES, PASSES = RB / ROWS;
    static_assert(RB % ROWS == 0, "passes");
    const int lane = threadIdx.x & 63, row = lane / LANES, cc = lane % LANES * 8, c = c0 + cc;
    const float* p = ep + row * LD + (GATED ? (cc >> 4) * 32 + (cc & 15) : cc);
    const bool whole = d.vector && c0 + COLS <= d.n, add = d.residual && whole;
    const auto ask = [&](int i) {
        return load_eight(d.residual, d.residual_type, (size_t)min(r0 + row + ROWS * i, d.rows - 1) * d.residual_stride + c);
    };
    if (!GATED && whole && !d.bias && d.act == ACT_NONE) {
        Eight res[PASSES];
        if (add) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) res[i] = ask(i);
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = r0 + row + ROWS * i;
            f8_t v = *reinterpret_cast<const f8_t*>(p + i * ROWS * LD);
            if (add) v += values(res[i], d.residual_type);
            if (r < d.rows) store_eight(d.out, d.out_type, (size_t)r * d.out_stride + c, v);
        }
        return;
    }
    f8_t bias = {0, 0, 0, 0, 0, 0, 0, 0}, bias_up = bias;
    if (d.bias && whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            bias[j] = load_one(d.bias, d.bias_type, c + j);
            if constexpr (GATED) bias_up[j] = load_one(d.bias, d.bias_type, (size_t)d.n + c + j);
        }
    }
    Eight res{}, next{};
    if (add) res = ask(0);
#pragma unroll 1
    for (int i = 0; i < PASSES; ++i, p += ROWS * LD, res = next) {
        const int r = r0 + row + ROWS * i;
        if (add && i + 1 < PASSES) next = ask(i + 1);
        f8_t v = *reinterpret_cast<const f8_t*>(p), up = v;
        if constexpr (GATED) up = *reinterpret_cast<const f8_t*>(p + 16);
        if (whole) {
            v += bias;
            if constexpr (GATED) up += bias_up;
            v = shape<GATED>(v, up, d.act, d.limit);
            if (add) v += values(res, d.residual_type);
            if (r < d.rows) store_eight(d.out, d.out_type, (size_t)r * d.out_stride + c, v);
        } else if (r < d.rows) {
            finish_some<GATED, 8>(d, r, c, v, up);
        }
    }
}

// Row of w for row i of a tile whose first output column is c0 (rows past the end: the last one, not stored).
template <bool GATED>
__device__ __forceinline__ int weight_row(const DenseJob& d, int c0, int i) {
    if constexpr (GATED) return min(c0 + (i >> 5) * 16 + (i & 15), d.n - 1) + ((i >> 4) & 1) * d.n;
    return min(c0 + i, d.n - 1);
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
// Needs a tile's rows within 32-bit offsets. DIRECT: the loads go straight to LDS, for 16-byte aligned rows; others go
// through registers. k past the last multiple of 64 is staged element by element (load_chunk), so that nothing beyond k
// is read.
// Bound, large: the matrix core at the clock that full load leaves (8192 rows, 5120 -> 2 x 12288 gated 1470 us, 12288 ->
// 5120 783 us: 1402 and 1317 TFLOP/s, where a library's product of 8192^3 runs at 1347). One round of 128 x 128 tiles: the
// tiles' way from L2 (709 x 5120 x 12288 in 117 us; in copies for timing only, every step's loads from the same lines, in
// L2, take 102, no loads 77, one fragment read of six 106): 32 KB a step and CU, 12.6 TB/s over the card. A larger tile asks for
// less, and leaves CUs without one. A stage more or less, four waves instead of eight, waves of 32 x 64 instead of 64 x
// 32, a barrier that waits for no reads and scalar-only addresses measured the same; with a step's loads in one burst the
// first form of the 256 x 256 tiles took 1641 us of the gated product above.
template <bool GATED, int NT, int RT, int WN, int WR, int NSA, int NSB>
struct TileShape {
    static constexpr int COLS = GATED ? NT / 2 : NT;               // columns of out
    static constexpr int WAVES = WN * WR, THREADS = 64 * WAVES;
    static constexpr int STAGE_A = NT * 128, STAGE_B = RT * 128, B0 = NSA * STAGE_A;
    static constexpr int MA = NT / WN / 16, NB = RT / WR / 16, LA = NT / 8 / WAVES, LB = RT / 8 / WAVES;
    // the epilogue's transposition: up to 64 rows of a wave's columns in fp32, padded by 4
    static constexpr int EP_ROWS = RT / WR < 64 ? RT / WR : 64, EP_LD = NT / WN + 4, EP_WAVE = EP_ROWS * EP_LD * 4;
    static constexpr int STAGES = B0 + NSB * STAGE_B;
    static constexpr int LDS = STAGES > WAVES * EP_WAVE ? STAGES : WAVES * EP_WAVE;
    // this wave's loads that may be in flight when a step's have to have landed
    static constexpr int AHEAD = (NSA - 2) * LA + (NSB - 2) * LB;
    static_assert(NT % (8 * WAVES) == 0 && RT % (8 * WAVES) == 0 && NT % (32 * WN) == 0 && RT % (16 * WR) == 0, "tile");
    static_assert(NSB >= 2 && (NSA == NSB || NSA == NSB + 1) && LDS <= 163840, "stages");
};

template <int TYPE, bool GATED, bool DIRECT, int NT, int RT, int WN, int WR, int NSA, int NSB>
__global__ void __launch_bounds__(64 * WN * WR) dense_tile_kernel(DenseJob d) {
    using S = TileShape<GATED, NT, RT, WN, WR, NSA, NSB>;
    extern __shared__ __align__(1024) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), a = lane & 15, q = lane >> 4;
    int tn, tr;
    tile_of(d, blockIdx.x, tn, tr);
    const int c0 = tn * S::COLS, r0 = tr * RT;

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
    // A half step (32 k): its MFMAs on the fragments in hand, and between equal shares of the first three quarters of
    // them the reads of the next half's fragments and `loads` direct loads, one by one. In this order and no other: a
    // wave issues in order, so that a burst of loads would hold back its MFMAs until the address units have taken them
    // (16 cycles each, eight waves' worth of them).
    auto half = [&](const uint4 (&ca)[S::MA], const uint4 (&cb)[S::NB], uint4 (&na)[S::MA], uint4 (&nb)[S::NB], int sa, int sb,
                    int s, auto loads, auto&& load) {
        constexpr int READS = S::MA + S::NB, MFMAS = S::MA * S::NB, SPREAD = MFMAS * 3 / 4, L = decltype(loads)::value;
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            read_one(i, sa, sb, s, na, nb);
#pragma unroll
            for (int j = (i * L + READS - 1) / READS; j < ((i + 1) * L + READS - 1) / READS; ++j) load(j);
#pragma unroll
            for (int f = i * SPREAD / READS; f < (i + 1) * SPREAD / READS; ++f)
                acc[f / S::NB][f % S::NB] = mfma<TYPE>(ca[f / S::NB], cb[f % S::NB], acc[f / S::NB][f % S::NB]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int f = SPREAD; f < MFMAS; ++f)
            acc[f / S::NB][f % S::NB] = mfma<TYPE>(ca[f / S::NB], cb[f % S::NB], acc[f / S::NB][f % S::NB]);
        __builtin_amdgcn_sched_barrier(0);
    };

    // A step's first half loads the weights of step t + NSA - 1 (to the place of step t - 1), its second half the rows of
    // step t + NSB (to its own place). Between the halves every wave's reads of step t are done, and its loads of step
    // t + 1 have landed (loads land in order).
    uint4 a0[S::MA], b0[S::NB], a1[S::MA], b1[S::NB];
    // k past the last multiple of 64, before the rest (after it, the compiler kept a second copy of the sums)
    if (d.k % 64) {
#pragma unroll 1
        for (int i = threadIdx.x; i < (NT + RT) * 8; i += S::THREADS) {
            const int row = i >> 3, c = i & 7;
            const uint16_t* p = row < NT ? d.w + (size_t)weight_row<GATED>(d, c0, row) * d.w_stride
                                         : d.x + (size_t)min(r0 + row - NT, d.rows - 1) * d.x_stride;
            char* to = row < NT ? lds + row * 128 : lds + S::B0 + (row - NT) * 128;
            *reinterpret_cast<uint4*>(to + (c ^ (row & 7)) * 16) = load_chunk(p, steps * 64 + c * 8, d.k);
        }
        lds_barrier();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int i = 0; i < S::MA + S::NB; ++i) read_one(i, 0, 0, s, a0, b0);
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
#pragma unroll
                for (int n = 0; n < S::NB; ++n) acc[m][n] = mfma<TYPE>(a0[m], b0[n], acc[m][n]);
        }
        lds_barrier();
    }
    if constexpr (DIRECT) {
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
    } else if (steps > 0) {
        // Through registers, two stages: step t + 2's values are asked for in step t's first half and go to step t's place
        // after its second (a step past the end is the last one again, and not read).
        static_assert(DIRECT || (NSA == 2 && NSB == 2), "two stages");
        uint4 rw[S::LA + S::LB];
        auto ask = [&](int j, int step) {
            const uint64_t base = j >= S::LA ? xbase : GATED && ((wave * S::LA + j) * 8 & 16) ? ubase : wbase;
            uint4 v;
            __builtin_memcpy(&v, reinterpret_cast<const char*>(base + (uint64_t)min(step, steps - 1) * 128) +
                                     (j >= S::LA ? vb[j >= S::LA ? j - S::LA : 0] : va[j >= S::LA ? 0 : j]), 16);
            rw[j] = v;
        };
        auto put = [&](int stage) {
#pragma unroll
            for (int j = 0; j < S::LA; ++j)
                *reinterpret_cast<uint4*>(lds + stage * S::STAGE_A + (wave * S::LA + j) * 1024 + lane * 16) = rw[j];
#pragma unroll
            for (int j = 0; j < S::LB; ++j)
                *reinterpret_cast<uint4*>(lds + S::B0 + stage * S::STAGE_B + (wave * S::LB + j) * 1024 + lane * 16) = rw[S::LA + j];
        };
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int j = 0; j < S::LA + S::LB; ++j) ask(j, p);
            put(p);
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < S::MA + S::NB; ++i) read_one(i, 0, 0, 0, a0, b0);
        for (int t = 0; t < steps; ++t) {
            half(a0, b0, a1, b1, t & 1, t & 1, 1, std::integral_constant<int, S::LA + S::LB>{}, [&](int j) { ask(j, t + 2); });
            lds_barrier();
            half(a1, b1, a0, b0, (t + 1) & 1, (t + 1) & 1, 0, std::integral_constant<int, 0>{}, [](int) {});
            put(t & 1);
        }
    }
    // Epilogue, through the wave's part of LDS
    lds_barrier();
    float* ep = reinterpret_cast<float*>(lds + wave * S::EP_WAVE);
#pragma unroll
    for (int n = 0; n < S::NB; n += S::EP_ROWS / 16) {
#pragma unroll
        for (int h = 0; h < S::EP_ROWS / 16; ++h)
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
                *reinterpret_cast<f4_t*>(ep + (16 * h + a) * S::EP_LD + 16 * m + 4 * q) = acc[m][n + h];
        __builtin_amdgcn_wave_barrier();
        finish_rows<GATED, S::COLS / WN, S::EP_ROWS, S::EP_LD>(d, ep, r0 + wr * (RT / WR) + 16 * n, c0 + wn * (S::COLS / WN));
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- few rows -------------------------------------------------------------------------------------------------------
// A workgroup owns `cols` columns of out and 16 RB rows over the whole K; its WAVES waves take the 64-k chunks in turn,
// each with all of the columns and rows, and their sums meet in LDS, added in wave order. A wave loads whole lines (8
// lanes of 16 bytes a row: loads in the fragments' own layout, whose neighbouring lanes are different rows, ran at 16
// bytes a cycle and CU), turns them into fragments through a stage of its own in LDS (the swizzle of the tiles; no
// barrier, a wave's LDS operations complete in order), and has the next U chunks' loads in flight meanwhile.
// Bound: HBM (weights out of the caches; the same read by a library's product in brackets): 1 row, 5120 -> 2 x 12288
// gated 45.4 us, 5540 GB/s (49.8); 12288 -> 5120 26.6 us, 4723 GB/s (29.2); 16 rows of it 28.0 (31.1); 5120^2 12.5 us,
// 4185 GB/s (13.4), where a round's start and end show.
// EB tiles of 16 weight rows hold the columns: CC = 16 a tile, or 8 gate rows and the 8 up rows of the same columns. With
// fewer than EB CC columns the last are read twice and dropped: `cols` is chosen so that every CU gets as much work.
template <int TYPE, bool GATED, int EB, int RB, int WAVES, int U>
__global__ void __launch_bounds__(64 * WAVES) dense_thin_kernel(DenseJob d) {
    constexpr int CC = GATED ? 8 : 16, TILES = EB + RB, STAGE = TILES * 2048;
    extern __shared__ __align__(1024) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, a = lane & 15, q = lane >> 4;
    int tn, tr;
    tile_of(d, blockIdx.x, tn, tr);
    const int c0 = tn * d.cols, c1 = min(c0 + d.cols, d.n) - 1, r0 = tr * 16 * RB;
    // this lane's 16 bytes of every 8 rows of a chunk
    const uint16_t *wp[2 * EB], *xp[2 * RB];
    bool xl[2 * RB];
#pragma unroll
    for (int i = 0; i < 2 * EB; ++i) {
        const int e = 8 * i + (lane >> 3);
        const int row = GATED ? min(c0 + (i >> 1) * 8 + (lane >> 3), c1) + (i & 1) * d.n : min(c0 + e, c1);
        wp[i] = d.w + (size_t)row * d.w_stride + (lane & 7) * 8;
    }
#pragma unroll
    for (int i = 0; i < 2 * RB; ++i) {
        const int row = r0 + 8 * i + (lane >> 3);
        xl[i] = row < d.rows;
        xp[i] = d.x + (size_t)min(row, d.rows - 1) * d.x_stride + (lane & 7) * 8;
    }
    char* stage = lds + wave * STAGE;
    char* to = stage + (lane >> 3) * 128 + ((lane & 7) ^ (lane >> 3)) * 16;
    const char* from = stage + a * 128;
    f4_t acc[EB][RB];
#pragma unroll
    for (int i = 0; i < EB; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j) acc[i][j] = (f4_t){0.f, 0.f, 0.f, 0.f};
    const int chunks = (d.k + 63) / 64;
    struct Chunk {
        uint4 w[2 * EB], x[2 * RB];
    };
    auto load = [&](Chunk& f, int c) {
        const int k = c * 64;
        if (k + 64 <= d.k) {
#pragma unroll
            for (int i = 0; i < 2 * EB; ++i) __builtin_memcpy(&f.w[i], wp[i] + k, 16);
#pragma unroll
            for (int i = 0; i < 2 * RB; ++i) {
                f.x[i] = make_uint4(0, 0, 0, 0);
                if (xl[i]) __builtin_memcpy(&f.x[i], xp[i] + k, 16);
            }
        } else {
            const int left = d.k - k - (lane & 7) * 8;             // from this lane's first on; nothing past the end
#pragma unroll
            for (int i = 0; i < 2 * EB; ++i) f.w[i] = load_chunk(wp[i] + k, 0, left);
#pragma unroll
            for (int i = 0; i < 2 * RB; ++i) f.x[i] = load_chunk(xp[i] + k, 0, left);
        }
    };
    auto multiply = [&](const Chunk& f) {
#pragma unroll
        for (int i = 0; i < 2 * EB; ++i) *reinterpret_cast<uint4*>(to + i * 1024) = f.w[i];
#pragma unroll
        for (int i = 0; i < 2 * RB; ++i) *reinterpret_cast<uint4*>(to + (2 * EB + i) * 1024) = f.x[i];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int at = ((4 * s + q) ^ (a & 7)) * 16;
            uint4 fw[EB], fx[RB];
#pragma unroll
            for (int i = 0; i < EB; ++i) fw[i] = *reinterpret_cast<const uint4*>(from + i * 2048 + at);
#pragma unroll
            for (int j = 0; j < RB; ++j) fx[j] = *reinterpret_cast<const uint4*>(from + (EB + j) * 2048 + at);
#pragma unroll
            for (int j = 0; j < RB; ++j)
#pragma unroll
                for (int i = 0; i < EB; ++i) acc[i][j] = mfma<TYPE>(fw[i], fx[j], acc[i][j]);
        }
        __builtin_amdgcn_wave_barrier();
    };
    // U chunks in flight: chunk c + U WAVES is asked for when chunk c is used
    Chunk f[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (wave + u * WAVES < chunks) load(f[u], wave + u * WAVES);
    for (int c = wave; c < chunks; c += U * WAVES) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (c + u * WAVES < chunks) multiply(f[u]);
            if (c + (u + U) * WAVES < chunks) load(f[u], c + (u + U) * WAVES);
        }
    }
    __syncthreads();
    f4_t* part = reinterpret_cast<f4_t*>(lds);                     // [WAVES][EB * RB][64]
#pragma unroll
    for (int i = 0; i < EB; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j) part[(wave * EB * RB + i * RB + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // a thread finishes four columns of a row: lane 16 Q + (row) of a tile holds columns 4 Q .. (a gated tile's up values
    // are two quads further on)
    constexpr int QUADS = CC / 4;
#pragma unroll 1
    for (int t = threadIdx.x; t < EB * RB * QUADS * 16; t += 64 * WAVES) {
        const int row = t & 15, Q = (t >> 4) % QUADS, tile = (t >> 4) / QUADS, i = tile / RB, j = tile % RB;
        const int r = r0 + 16 * j + row, col = c0 + CC * i + 4 * Q;
        if (r >= d.rows || col > c1) continue;
        f8_t v = {0, 0, 0, 0, 0, 0, 0, 0}, up = v;
#pragma unroll
        for (int s = 0; s < WAVES; ++s) {
            const f4_t* p = part + (s * EB * RB + tile) * 64 + 16 * Q + row;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += p[0][e];
            if constexpr (GATED) {
#pragma unroll
                for (int e = 0; e < 4; ++e) up[e] += p[32][e];
            }
        }
        finish_some<GATED, 4>(d, r, col, v, up);
    }
}

// ---- which form -----------------------------------------------------------------------------------------------------
// Every form is a workgroup of `cols` weight rows x `rows` rows over the whole K, so a call's time is its rounds of one
// workgroup a CU, each a fixed part and a time per 64 k that grows with the share of the CUs in use (they share the
// caches). Light and full: a chunk's time with few and with all CUs at work, us; fixed: a round's start and epilogue.
// Fitted to 190 sizes (rows 1 to 4096, 512 to 24576 weight rows, k 1024 to 12288, weights out of the caches), where the
// form this picks takes 1.015 times the fastest one's time on average, 1.25 at worst; rows off 16-byte alignment to 55 of
// their own (k 1001 to 8191), 1.014 and 1.45. 64 x 128, added to the others, to 84 and 40 (1.002 and 1.08, 1.002 and
// 1.03); of 85 and 40 other sizes it made 18 and 8 faster by 5 to 27 %, none slower by more than 4.5 %.
// Times of the forms in this order (us, bf16, plain form; -: not measured):
//   rows    n     k     16x16  32x16  32x32  32x64  64x64  64x128  128x128  128x256  256x256
//      1   4096  4096     9.8   10.4   11.1   13.7   18.2     -        -        -        -
//     16   5120 12288    34.5   27.8   29.2   35.4   46.2     -        -        -        -
//     64   4096  4096    20.3   16.7   14.7   18.0   20.8   23.8     33.1     47.4     82.2
//    128   5120  1536      -    16.1   13.5   15.4   11.1   11.7     19.2     23.1     37.7
//    384   5120  5120      -      -      -      -    51.8   39.1     51.0       -        -
//   1536   1024  4096      -      -      -      -    37.0   25.5     30.8       -        -
//    512   4096  4096      -      -    58.0   58.4   38.8   31.5     38.4     53.6     86.2
//   1536   4096  4096      -      -      -      -      -      -      71.2     58.1     86.3
//   4096  16384  2048      -      -      -      -      -      -     360.4    285.8    227.1
struct Form {
    int cols, rows;
    float light, full, fixed;
};
// and off alignment, the tiles through registers:
//     12   4099  4099    18.1   16.1   17.0   19.1   28.0     -        -        -
//    128   8191  2047    64.8   57.3   36.6   36.8   29.4     -      48.3     66.0
//    375   5113  4093      -      -      -      -    74.1   59.3     75.3       -
//   2492    506  4091      -      -      -      -    66.2   45.1     54.3       -
//    512   4099  4099      -      -   103.6  106.1   89.1     -      71.8    104.1
//   2000   8191  2047      -      -      -      -      -      -     146.7    134.5
constexpr Form ALIGNED[] = {{16, 16, .056f, .11f, .3f},     {32, 16, .075f, .136f, .4f},     {32, 32, .10f, .18f, .5f},
                            {32, 64, .135f, .237f, .7f},    {64, 64, .20f, .275f, 1.2f},     {64, 128, .207f, .406f, 2.4f},
                            {128, 128, .3625f, .53f, 2.2f}, {128, 256, .615f, .90f, 3.3f},   {256, 256, 1.017f, 1.5f, 5.5f}};
constexpr Form UNALIGNED[] = {{16, 16, .067f, .14f, .3f},  {32, 16, .091f, .22f, .4f}, {32, 32, .112f, .25f, .5f},
                              {32, 64, .153f, .42f, .7f},  {64, 64, .22f, .5f, 1.2f},  {64, 128, .41f, .571f, 6.7f},
                              {128, 128, .71f, .92f, 5.f}, {128, 256, 1.14f, 1.7f, 7.f}};
constexpr int THIN_FORMS = 5;                                      // the first ones: dense_thin_kernel
constexpr int CUS = 256;

// Columns a workgroup of a thin form: as many as it holds, evened out over whole rounds of one workgroup a CU.
int thin_cols(int n, int row_tiles, int most) {
    const int64_t tiles = (int64_t)((n + most - 1) / most) * row_tiles, rounds = (tiles + CUS - 1) / CUS;
    const int64_t per = rounds * CUS / row_tiles > 0 ? rounds * CUS / row_tiles : 1;
    const int cols = (int)((n + per - 1) / per + 3) / 4 * 4;
    return cols < most ? cols : most;
}
int pick_form(const DenseJob& d, bool aligned, bool tiles_fit) {
    int best = 0;
    double least = 0.;
    for (int f = 0; f < (!tiles_fit ? THIN_FORMS : aligned ? 9 : 8); ++f) {
        const Form& o = aligned ? ALIGNED[f] : UNALIGNED[f];
        const int row_tiles = (d.rows + o.rows - 1) / o.rows, most = d.gated ? o.cols / 2 : o.cols;
        const int cols = f < THIN_FORMS ? thin_cols(d.n, row_tiles, most) : most;
        const int64_t groups = (int64_t)((d.n + cols - 1) / cols) * row_tiles;
        const double chunks = (d.k + 63) / 64, part = (double)(groups % CUS) / CUS;
        const double t = (double)(groups / CUS) * (chunks * o.full + o.fixed) +
                         (part > 0. ? chunks * (o.light + (o.full - o.light) * part) + o.fixed : 0.);
        if (f == 0 || t < least) best = f, least = t;
    }
    return best;
}

bool multiple(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <int TYPE, bool GATED, bool DIRECT, int NT, int RT, int WN, int WR, int NSA, int NSB>
hipError_t launch_tile(hipStream_t s, DenseJob d) {
    using S = TileShape<GATED, NT, RT, WN, WR, NSA, NSB>;
    d.n_tiles = (d.n + S::COLS - 1) / S::COLS;
    const int64_t tiles = (int64_t)d.n_tiles * ((d.rows + RT - 1) / RT);
    dense_tile_kernel<TYPE, GATED, DIRECT, NT, RT, WN, WR, NSA, NSB><<<dim3((unsigned)tiles), S::THREADS, S::LDS, s>>>(d);
    return hipGetLastError();
}

template <int TYPE, bool GATED, int EB, int RB, int WAVES, int U>
hipError_t launch_thin(hipStream_t s, DenseJob d) {
    constexpr int PART = WAVES * EB * RB * 1024, STAGES = WAVES * (EB + RB) * 2048;
    const int row_tiles = (d.rows + 16 * RB - 1) / (16 * RB);
    d.cols = thin_cols(d.n, row_tiles, (GATED ? 8 : 16) * EB);
    d.n_tiles = (d.n + d.cols - 1) / d.cols;
    dense_thin_kernel<TYPE, GATED, EB, RB, WAVES, U>
        <<<dim3((unsigned)((int64_t)d.n_tiles * row_tiles)), 64 * WAVES, PART > STAGES ? PART : STAGES, s>>>(d);
    return hipGetLastError();
}

// the tiles take rows directly to LDS at 16-byte aligned addresses, and a tile's rows within 32-bit offsets
bool aligned_rows(const DenseJob& d) {
    return multiple(d.x, 16) && multiple(d.w, 16) && d.x_stride % 8 == 0 && d.w_stride % 8 == 0;
}
int form_of(const DenseJob& d, bool aligned) { return pick_form(d, aligned, d.x_stride < 1 << 22 && d.w_stride < 1 << 22); }

template <int TYPE, bool GATED>
hipError_t launch(hipStream_t s, DenseJob d) {
    const bool aligned = aligned_rows(d);
    switch (form_of(d, aligned)) {
        case 0: return launch_thin<TYPE, GATED, 1, 1, 8, 2>(s, d);
        case 1: return launch_thin<TYPE, GATED, 2, 1, 8, 2>(s, d);
        case 2: return launch_thin<TYPE, GATED, 2, 2, 8, 2>(s, d);
        case 3: return launch_thin<TYPE, GATED, 2, 4, 8, 2>(s, d);
        case 4: return launch_thin<TYPE, GATED, 4, 4, 8, 1>(s, d);
        case 5:
            return aligned ? launch_tile<TYPE, GATED, true, 64, 128, 2, 4, 5, 5>(s, d)
                           : launch_tile<TYPE, GATED, false, 64, 128, 2, 4, 2, 2>(s, d);
        case 6:
            return aligned ? launch_tile<TYPE, GATED, true, 128, 128, 2, 4, 4, 4>(s, d)
                           : launch_tile<TYPE, GATED, false, 128, 128, 2, 4, 2, 2>(s, d);
        case 7:
            return aligned ? launch_tile<TYPE, GATED, true, 128, 256, 2, 4, 3, 3>(s, d)
                           : launch_tile<TYPE, GATED, false, 128, 256, 2, 4, 2, 2>(s, d);
        default: return launch_tile<TYPE, GATED, true, 256, 256, 4, 2, 3, 2>(s, d);
    }
}

}  // namespace

int dense_form(const DenseJob& d) {
    const bool aligned = aligned_rows(d);
    return form_of(d, aligned) + (aligned ? 0 : 16);
}

hipError_t launch_dense(hipStream_t s, DenseJob d) {
    const auto eight = [](const void* p, int type, int64_t stride) {
        return !p || (stride % (type == TYPE_F32 ? 4 : 8) == 0 && multiple(p, 16));
    };
    d.vector = eight(d.out, d.out_type, d.out_stride) && eight(d.residual, d.residual_type, d.residual_stride);
    if (d.type == TYPE_BF16)
        return d.gated ? launch<TYPE_BF16, true>(s, d) : launch<TYPE_BF16, false>(s, d);
    return d.gated ? launch<TYPE_F16, true>(s, d) : launch<TYPE_F16, false>(s, d);
}

}  // namespace gfr
