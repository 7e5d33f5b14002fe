// 16-bit routed experts for a few tokens: with e = picks[r][s] the expert of pair (r, s),
//   g, u   = the halves of gu[e] x[r];  a = act(min(g, limit)) * clamp(u, -limit, limit)
//   out[r] = residual[r] + sum over s of weights[r][s] * down[e] a       (slots in order; picks outside [0, experts): none)
// x, gu and down in bf16 or fp16; sums, activations and weights in fp32, one rounding at the end. Between the two products
// the activations are held as two 16-bit values, which costs the matrix core a second pass over the same weights in
// registers: as h + l in bf16, 16 bits of them; as 2 h + l / 1024 in fp16, 22 bits or 2^-35 where that is more, up to twice its
// range. (2 h leaves 2^-11 of an activation or 2^-24, so that l is in range, and most of what is below fp16's least values is in
// it; with h + l that was lost, 2^-25, which left 12 bits of 1e-4.) The two parts' sums meet once a chunk.
//
// Bound: HBM, the weights of the experts that are picked, read once. A workgroup takes one expert's share of the columns and
// all the rows that picked it, in passes of up to 16 RB, so that an expert's weights are read once however many rows pick it
// (again, from the caches, for more than one pass). Weights are the matrix core's A operand (v_mfma_f32_16x16x32: D holds,
// in lane l, columns 4 (l / 16) .. + 3 of the tile for row l % 16) and go through LDS stages of a wave's own as whole lines;
// rows are the B operand, loaded as fragments, which the caches hold. A row's sums are taken in an order of the
// sizes alone, so that they depend neither on the other rows nor on their number.
// Graph replays, us (GB/s of weights): 64 rows top-8 of 160, 5120 -> 1408 bf16 1110 (5880); 12 rows top-8 of 288, 4096 ->
// 512 148 (6020); 4 rows top-8 of 64, 4096 -> 1024 115 (5800); one row of 9 slots, 4096 -> 512 28.8 (3930), where two launches'
// starts and ends are a quarter; 5 rows top-3 of 20, 1001 -> 333 fp16 19.6, all of it latency. Asking for the down matrices
// from the first launch's end made the one row slower (34 us).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lanes.hpp"
#include "launch.hpp"
#include "mfma16.hpp"
#include "values.hpp"

namespace gfr {
namespace {

constexpr int PASS = 64;                                             // a pass's members at most

// What an activation's two parts are in units of.
template <int TYPE>
constexpr float HIGH = TYPE == TYPE_BF16 ? 1.f : 2.f;
template <int TYPE>
constexpr float LOW = TYPE == TYPE_BF16 ? 1.f : 1.f / 1024;

// The members of an expert: the pairs (by number) whose pick it is, in order; first and their count over all, and those from
// number `from` on, up to `room` of them, in LDS. Called by the whole workgroup (waves of it, at most 16).
struct Members {
    int pair[PASS];
    int waves[16];
};
__device__ __forceinline__ int find_members(const Experts16Job& d, int expert, int from, int room, Members& m, int& first) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, pairs = d.rows * d.slots;
    int seen = 0;
    first = pairs;
    if (pairs <= 64) {                                                // each wave by itself, all with the same values
        const bool mine = lane < pairs && d.picks[lane] == expert;
        const uint64_t ballot = __ballot(mine);
        const int at = set_before(ballot) - from;
        if (mine && at >= 0 && at < room) m.pair[at] = lane;
        if (ballot) first = __builtin_ctzll(ballot);
        __builtin_amdgcn_wave_barrier();
        return __popcll(ballot);
    }
    for (int base = 0; base < pairs; base += blockDim.x) {
        const int p = base + (int)threadIdx.x;
        const bool mine = p < pairs && d.picks[p] == expert;
        const uint64_t ballot = __ballot(mine);
        __syncthreads();
        if (lane == 0) m.waves[wave] = __popcll(ballot);
        __syncthreads();
        int before = seen + set_before(ballot);
        for (int w = 0; w < waves; ++w) {
            if (w < wave) before += m.waves[w];
            seen += m.waves[w];
        }
        if (mine && before >= from && before < from + room) m.pair[before - from] = p;
    }
    __syncthreads();
    if (seen && from == 0) first = m.pair[0];
    return seen;
}

// This workgroup's expert: the experts in turn, or, where there are fewer pairs, the pairs' picks, each taken by the first
// pair that has it. Negative: nothing to do. count: its members; the first `room` are in LDS.
__device__ __forceinline__ int expert_of(const Experts16Job& d, int u, int room, Members& m, int& count) {
    const bool by_pair = d.rows * d.slots < d.experts;
    const int e = by_pair ? d.picks[u] : u;
    if (e < 0 || e >= d.experts) return -1;
    int first;
    count = find_members(d, e, 0, room, m, first);
    return count && (!by_pair || first == u) ? e : -1;
}

// A wave's stage of EB tiles of 16 weight rows by 64 k: rows of 128 bytes, 16-byte chunk c at position c ^ (row % 8), so
// that the fragments' reads of neighbouring rows meet all banks.
template <int TYPE, int EB>
struct Weights {
    const uint16_t* row[2 * EB];                                      // this lane's row of every eight
    struct Chunk {
        uint4 w[2 * EB];
    };
    // columns k .. + 63 of rows of K, at least eight: to be settled where K ends among them
    __device__ __forceinline__ void ask(Chunk& f, int k, int K) const {
        k += (threadIdx.x & 7) * 8;
#pragma unroll
        for (int i = 0; i < 2 * EB; ++i) f.w[i] = gfr::ask(row[i], k, K);
    }
    __device__ __forceinline__ void settle(Chunk& f, int k, int K) const {
        k += (threadIdx.x & 7) * 8;
#pragma unroll
        for (int i = 0; i < 2 * EB; ++i) f.w[i] = gfr::settle(f.w[i], k, K);
    }
    // rows of less than eight
    __device__ __forceinline__ void load_short(Chunk& f, int K) const {
#pragma unroll
        for (int i = 0; i < 2 * EB; ++i) f.w[i] = gfr::load_short(row[i], (threadIdx.x & 7) * 8, K);
    }
    __device__ __forceinline__ void stage(const Chunk& f, char* stage) const {
        const int lane = threadIdx.x & 63;
        char* to = stage + (lane >> 3) * 128 + ((lane & 7) ^ (lane >> 3)) * 16;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 2 * EB; ++i) *reinterpret_cast<uint4*>(to + i * 1024) = f.w[i];
        __builtin_amdgcn_wave_barrier();
    }
    // tile i's fragment of half s of the chunk: row l % 16, k 32 s + 8 (l / 16) ..
    __device__ __forceinline__ uint4 fragment(const char* stage, int i, int s) const {
        const int lane = threadIdx.x & 63, a = lane & 15, q = lane >> 4;
        return *reinterpret_cast<const uint4*>(stage + i * 2048 + a * 128 + ((4 * s + q) ^ (a & 7)) * 16);
    }
};

// U chunks in flight: f[u] of the n that this wave takes is used and asked for again U further on. Past the end the last one
// is asked for once more (the caches have it): a load under a condition would have the compiler wait for all loads wherever
// it cannot tell how many there are.
template <int U, typename Chunk, typename Load, typename Use>
__device__ __forceinline__ void pipeline(Chunk (&f)[U], int n, Load load, Use use) {
    if (n <= 0) return;
#pragma unroll
    for (int u = 0; u < U; ++u) load(f[u], min(u, n - 1));
    for (int i = 0; i < n; i += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u < n) use(f[u], i + u);
            load(f[u], min(i + u + U, n - 1));
        }
    }
}

// ---- gate and up --------------------------------------------------------------------------------------------------
// Eight waves (16 took 37.7 us and not 31.9 at one row, 1806 and not 1107 at 64), two chunks in flight (four: 34.1 and 1171; no
// registers for them). Two tiles a wave, and one where the workgroups would be fewer than 1.25 a CU: one row of 9 slots, 4096
// -> 512 29.3 us and not 31.5, 4 rows of 2, 1024 -> 256 9.3 and 9.6; beyond that 2 rows of 8 43.0 and 41.8, 64 rows 1238 and 1110.
constexpr int UP_WAVES = 8;

// One pass: members [from, from + 16 RB) of the expert, columns c0 .. + 8 EB. A tile of 16 weight rows is 8 gate rows
// and the 8 up rows of the same columns; the waves share k by chunks of 64, and their sums are added in order.
template <int TYPE, int EB, int RB>
__device__ __forceinline__ void up_pass(const Experts16Job& d, const Weights<TYPE, EB>& w, const Members& m, int members,
                                        int c0, char* lds) {
    constexpr int U = 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), a = lane & 15, q = lane >> 4;
    const uint16_t* xp[RB];
#pragma unroll
    for (int j = 0; j < RB; ++j) {
        const int pair = m.pair[min(16 * j + a, members - 1)];
        xp[j] = d.x + (int64_t)(pair / d.slots) * d.x_stride;
    }
    struct Chunk {
        typename Weights<TYPE, EB>::Chunk w;
        uint4 x[RB][2];
    };
    f4_t acc[EB][RB];
#pragma unroll
    for (int i = 0; i < EB; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j) acc[i][j] = (f4_t){0.f, 0.f, 0.f, 0.f};
    const int K = d.hidden, chunks = (K + 63) / 64;
    auto load = [&](Chunk& f, int i) {
        const int k = (wave + i * UP_WAVES) * 64;
        w.ask(f.w, k, K);
#pragma unroll
        for (int j = 0; j < RB; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s) f.x[j][s] = ask(xp[j], k + 32 * s + 8 * q, K);
    };
    char* stage = lds + wave * EB * 2048;
    auto product = [&](const Chunk& f) {
        w.stage(f.w, stage);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < EB; ++i) {
                const uint4 fw = w.fragment(stage, i, s);
#pragma unroll
                for (int j = 0; j < RB; ++j) acc[i][j] = mfma<TYPE>(fw, f.x[j][s], acc[i][j]);
            }
    };
    auto multiply = [&](Chunk& f, int i) {
        const int k = (wave + i * UP_WAVES) * 64;
        if (k + 64 > K) {
            w.settle(f.w, k, K);
#pragma unroll
            for (int j = 0; j < RB; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s) f.x[j][s] = settle(f.x[j][s], k + 32 * s + 8 * q, K);
        }
        product(f);
    };
    Chunk f[U];
    if (K >= 8) {
        pipeline(f, (chunks - wave + UP_WAVES - 1) / UP_WAVES, load, multiply);
    } else if (wave == 0) {
        w.load_short(f[0].w, K);
#pragma unroll
        for (int j = 0; j < RB; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s) f[0].x[j][s] = load_short(xp[j], 32 * s + 8 * q, K);
        product(f[0]);
    }
    __syncthreads();
    f4_t* part = reinterpret_cast<f4_t*>(lds);                        // [UP_WAVES][EB * RB][64]
#pragma unroll
    for (int i = 0; i < EB; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j) part[(wave * EB * RB + i * RB + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // a thread finishes four columns of a member: lanes 16 Q + member hold gate columns 4 Q .., lanes 32 on their up values
    for (int t = threadIdx.x; t < EB * RB * 32; t += 64 * UP_WAVES) {
        const int row = t & 15, Q = (t >> 4) & 1, tile = t >> 5, i = tile / RB, j = tile % RB;
        if (16 * j + row >= members) continue;
        f8_t v = {0, 0, 0, 0, 0, 0, 0, 0}, up = v;
        for (int s = 0; s < UP_WAVES; ++s) {
            const f4_t* p = part + (s * EB * RB + tile) * 64 + 16 * Q + row;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += p[0][e], up[e] += p[32][e];
        }
        v = shape<true>(v, up, d.act, d.limit);
        const int col = c0 + 8 * i + 4 * Q;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = col + e < d.inter ? v[e] : 0.f;           // (columns up to a multiple of 64 are read)
            hi[e] = f_to_16(x / HIGH<TYPE>, TYPE);
            const float h = HIGH<TYPE> * (TYPE == TYPE_BF16 ? bf16_to_f(hi[e]) : f16_to_f(hi[e]));
            lo[e] = fabsf(h) < INFINITY ? f_to_16((x - h) / LOW<TYPE>, TYPE) : 0;
        }
        uint16_t* to = d.acts + (int64_t)m.pair[16 * j + row] * 2 * d.inter_pad + col;
        *reinterpret_cast<uint2*>(to) = make_uint2(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16);
        *reinterpret_cast<uint2*>(to + d.inter_pad) = make_uint2(lo[0] | lo[1] << 16, lo[2] | lo[3] << 16);
    }
    __syncthreads();
}

template <int TYPE, int EB, int RB>
__global__ void __launch_bounds__(64 * UP_WAVES, RB == 1 ? 4 : 2) experts16_up_kernel(Experts16Job d) {
    __shared__ __align__(1024) char lds[UP_WAVES * EB * (RB > 2 ? RB * 1024 : 2048)];
    __shared__ Members m;
    const int lane = threadIdx.x & 63, tiles = d.inter_pad / (8 * EB);
    const int u = blockIdx.x / tiles, c0 = (blockIdx.x % tiles) * 8 * EB;
    int count;
    const int e = expert_of(d, u, 16 * RB, m, count);
    if (e < 0) return;
    Weights<TYPE, EB> w;
#pragma unroll
    for (int i = 0; i < 2 * EB; ++i) {
        const int row = min(c0 + (i >> 1) * 8 + (lane >> 3), d.inter - 1) + (i & 1) * d.inter;
        w.row[i] = d.gu + (int64_t)e * d.gu_expert + (int64_t)row * d.gu_stride;
    }
    for (int from = 0;;) {
        const int members = min(count - from, 16 * RB);
        if constexpr (RB == 1) {
            up_pass<TYPE, EB, 1>(d, w, m, members, c0, lds);
        } else {
            if (members <= 16) up_pass<TYPE, EB, 1>(d, w, m, members, c0, lds);
            else if (members <= 32) up_pass<TYPE, EB, 2>(d, w, m, members, c0, lds);
            else up_pass<TYPE, EB, 4>(d, w, m, members, c0, lds);
        }
        if ((from += 16 * RB) >= count) break;
        int first;
        find_members(d, e, from, 16 * RB, m, first);
    }
}

// ---- down ---------------------------------------------------------------------------------------------------------
// (bounds of three waves a SIMD, 123 registers; held to four when it had 146, with registers spilled, 12 rows took 161 us and
// not 148)
constexpr int DOWN_WAVES = 4, DOWN_TILES = 2, DOWN_COLS = 16 * DOWN_TILES * DOWN_WAVES;

// A tile's sum over a chunk in units of HIGH, in an order that both forms of the product share (each adds the chunks' sums in
// turn).
template <int TYPE>
__device__ __forceinline__ f4_t chunk_sum(uint4 w0, uint4 w1, const uint4 (&x)[2][2]) {
    const f4_t none = {0.f, 0.f, 0.f, 0.f};
    if constexpr (LOW<TYPE> != HIGH<TYPE>) {
        f4_t high = mfma<TYPE>(w0, x[0][0], none), low = mfma<TYPE>(w0, x[0][1], none);
        high = mfma<TYPE>(w1, x[1][0], high), low = mfma<TYPE>(w1, x[1][1], low);
#pragma unroll
        for (int j = 0; j < 4; ++j) high[j] = fmaf(low[j], LOW<TYPE> / HIGH<TYPE>, high[j]);
        return high;
    }
    f4_t v = mfma<TYPE>(w0, x[0][0], none);
    v = mfma<TYPE>(w0, x[0][1], v);
    v = mfma<TYPE>(w1, x[1][0], v);
    return mfma<TYPE>(w1, x[1][1], v);
}

// One pass: a wave's 16 DOWN_TILES columns from c0 on, for members [from, from + 16 RB), over the whole of k.
template <int TYPE, int RB>
__device__ __forceinline__ void down_pass(const Experts16Job& d, const Weights<TYPE, DOWN_TILES>& w, const Members& m,
                                          int members, int c0, char* stage) {
    constexpr int EB = DOWN_TILES, U = RB == 4 ? 1 : 2;
    const int lane = threadIdx.x & 63, a = lane & 15, q = lane >> 4;
    const uint16_t* xp[RB];
#pragma unroll
    for (int j = 0; j < RB; ++j)
        xp[j] = d.acts + (int64_t)m.pair[min(16 * j + a, members - 1)] * 2 * d.inter_pad + 8 * q;
    struct Chunk {
        typename Weights<TYPE, EB>::Chunk w;
        uint4 x[RB][2][2];
    };
    f4_t acc[EB][RB];
#pragma unroll
    for (int i = 0; i < EB; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j) acc[i][j] = (f4_t){0.f, 0.f, 0.f, 0.f};
    const int K = d.inter, chunks = d.inter_pad / 64;
    auto load_rows = [&](Chunk& f, int c) {
#pragma unroll
        for (int j = 0; j < RB; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                f.x[j][s][0] = *reinterpret_cast<const uint4*>(xp[j] + c * 64 + 32 * s);
                f.x[j][s][1] = *reinterpret_cast<const uint4*>(xp[j] + d.inter_pad + c * 64 + 32 * s);
            }
    };
    auto load = [&](Chunk& f, int c) {
        w.ask(f.w, c * 64, K);
        load_rows(f, c);
    };
    auto product = [&](const Chunk& f) {
        w.stage(f.w, stage);
#pragma unroll
        for (int i = 0; i < EB; ++i) {
            const uint4 w0 = w.fragment(stage, i, 0), w1 = w.fragment(stage, i, 1);
#pragma unroll
            for (int j = 0; j < RB; ++j) acc[i][j] += chunk_sum<TYPE>(w0, w1, f.x[j]);
        }
    };
    auto multiply = [&](Chunk& f, int c) {
        if (c * 64 + 64 > K) w.settle(f.w, c * 64, K);
        product(f);
    };
    Chunk f[U];
    if (K >= 8) {
        pipeline(f, chunks, load, multiply);
    } else {
        w.load_short(f[0].w, K);
        load_rows(f[0], 0);
        product(f[0]);
    }
#pragma unroll
    for (int j = 0; j < RB; ++j) {
        if (16 * j + a >= members) continue;
        float* y = d.y + (int64_t)m.pair[16 * j + a] * d.hidden_pad;
#pragma unroll
        for (int i = 0; i < EB; ++i) {
            const int col = c0 + 16 * i + 4 * q;
            if (col < d.hidden) *reinterpret_cast<f4_t*>(y + col) = acc[i][j] * HIGH<TYPE>;
        }
    }
}

template <int TYPE, int RB>
__global__ void __launch_bounds__(64 * DOWN_WAVES, RB == 1 ? 3 : 2) experts16_down_kernel(Experts16Job d) {
    __shared__ __align__(1024) char lds[DOWN_WAVES * DOWN_TILES * 2048];
    __shared__ Members m;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tiles = (d.hidden + DOWN_COLS - 1) / DOWN_COLS;
    const int u = blockIdx.x / tiles, c0 = (blockIdx.x % tiles) * DOWN_COLS + wave * 16 * DOWN_TILES;
    int count;
    const int e = expert_of(d, u, 16 * RB, m, count);
    if (e < 0) return;
    Weights<TYPE, DOWN_TILES> w;
#pragma unroll
    for (int i = 0; i < 2 * DOWN_TILES; ++i)
        w.row[i] = d.down + (int64_t)e * d.down_expert + (int64_t)min(c0 + i * 8 + (lane >> 3), d.hidden - 1) * d.down_stride;
    char* stage = lds + wave * DOWN_TILES * 2048;
    for (int from = 0;;) {
        const int members = min(count - from, 16 * RB);
        if constexpr (RB == 1) {
            down_pass<TYPE, 1>(d, w, m, members, c0, stage);
        } else {
            if (members <= 16) down_pass<TYPE, 1>(d, w, m, members, c0, stage);
            else if (members <= 32) down_pass<TYPE, 2>(d, w, m, members, c0, stage);
            else down_pass<TYPE, 4>(d, w, m, members, c0, stage);
        }
        if ((from += 16 * RB) >= count) break;
        __syncthreads();                                              // (the waves are done with the last pass's members)
        int first;
        find_members(d, e, from, 16 * RB, m, first);
    }
}

// ---- the rows' sums -----------------------------------------------------------------------------------------------
// Up to four columns of a row with their residual.
__device__ __forceinline__ f4_t residual_at(const Experts16Job& d, int row, int col) {
    f4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (d.residual && col + j < d.hidden) v[j] = load_one(d.residual, d.residual_type, (int64_t)row * d.residual_stride + col + j);
    return v;
}
__device__ __forceinline__ void finish(const Experts16Job& d, int row, int col, f4_t v, f4_t residual) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (col + j < d.hidden)
            store_one(d.out, d.out_type, (int64_t)row * d.out_stride + col + j, d.residual ? v[j] + residual[j] : v[j]);
}
__global__ void __launch_bounds__(256) experts16_combine_kernel(Experts16Job d) {
    const int quads = d.hidden_pad / 4;
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (int64_t)d.rows * quads) return;
    const int row = (int)(t / quads), col = (int)(t % quads) * 4;
    const f4_t residual = residual_at(d, row, col);
    f4_t v = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < d.slots; s0 += 8) {                         // eight slots' loads at once
        f4_t y[8];
        float weight[8];
        bool there[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const int pair = row * d.slots + min(s0 + s, d.slots - 1), e = d.picks[pair];
            there[s] = s0 + s < d.slots && e >= 0 && e < d.experts;
            weight[s] = d.weights[pair];
            y[s] = *reinterpret_cast<const f4_t*>(d.y + (int64_t)pair * d.hidden_pad + col);
        }
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = there[s] ? fmaf(weight[s], y[s][j], v[j]) : v[j];
    }
    finish(d, row, col, v, residual);
}

// ---- down and the rows' sums at once, for few pairs ---------------------------------------------------------------
// A workgroup takes 16 columns of all pairs (inter at least 8): its waves share the picked experts' chunks of k in turn, a
// chunk's sums of its members go to LDS, and are added there in the order of the other form: chunks, then slots. Every wave lists the
// picks for itself, and few workgroups hold long chains of chunks, so that this is for up to 10 pairs and 96 chunks of them.
// us with it, and with the down launch and the rows' sums in another: 1 row of 9 slots, 4096 -> 512 28.8, 33.1; 1 of 4, 2048 ->
// 768 13.7, 16.4; 4 of 2, 1024 -> 256 8.7, 10.3; 1 of 8, 4097 -> 511 34.1, 34.7; and beyond: 1 of 8, 2048 -> 1024 29.6, 28.9; 5 of
// 3, 1024 -> 384 17.3, 15.4; 1 of 8, 7168 -> 2048 132, 127. (16 or 4 waves at the first: 34.2, 30.0; three chunks in flight 29.4.)
constexpr int FEW_WAVES = 8, FEW_PAIRS = 10, FEW_UNITS = 96;

template <int TYPE>
__global__ void __launch_bounds__(64 * FEW_WAVES) experts16_few_kernel(Experts16Job d) {
    constexpr int U = 2;
    __shared__ __align__(1024) char stages[FEW_WAVES * 2048];
    __shared__ f4_t parts[FEW_UNITS * 4], sums[FEW_PAIRS * 4];        // [pairs][chunks][4], [pairs][4]
    __shared__ float weight[FEW_PAIRS];                               // of the pairs, and whether an expert is theirs
    __shared__ bool there[FEW_PAIRS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), a = lane & 15, q = lane >> 4;
    const int c0 = blockIdx.x * 16, pairs = d.rows * d.slots, chunks = d.inter_pad / 64;
    char* stage = stages + wave * 2048;

    // the picked experts, one a lane, with the pairs that picked them
    const int pick = lane < pairs ? d.picks[lane] : -1;
    if (threadIdx.x < pairs) weight[threadIdx.x] = d.weights[threadIdx.x], there[threadIdx.x] = pick >= 0 && pick < d.experts;
    int expert = 0, count = 0;
    uint32_t members = 0;
    for (int i = 0; i < pairs; ++i) {
        const int e = __builtin_amdgcn_readlane(pick, i);
        const uint32_t same = (uint32_t)__ballot(pick == e && lane < pairs);
        if (e < 0 || e >= d.experts || __builtin_ctz(same) != i) continue;
        if (lane == count) expert = e, members = same;
        ++count;
    }
    const int units = count * chunks, my_row = threadIdx.x >> 2, my_col = c0 + (threadIdx.x & 3) * 4;
    f4_t residual = {0.f, 0.f, 0.f, 0.f};
    if (my_row < d.rows) residual = residual_at(d, my_row, my_col);   // (asked for ahead of its use)
    const int64_t row0 = min(c0 + (lane >> 3), d.hidden - 1), row1 = min(c0 + 8 + (lane >> 3), d.hidden - 1);
    struct Unit {
        typename Weights<TYPE, 1>::Chunk w;
        uint4 x[2][2];
        int pair;                                                     // this lane's member; negative: none
        int c;
    };
    // the n-th pair of a set, n = this lane's a; negative: there are fewer
    const auto nth = [&](uint32_t set) {
        if (!(set & (set - 1))) return a == 0 ? (int)__builtin_ctz(set) : -1;
        const bool in = lane < 32 && (set >> (lane & 31) & 1);
        const int list = __builtin_amdgcn_ds_permute((in ? set_before(set) : 63) * 4, lane);
        const int mine = __builtin_amdgcn_ds_bpermute(a * 4, list);
        return a < __popc(set) ? mine : -1;
    };
    // this wave's place among the units: expert n's chunk c, its weights and pairs; units are asked for in turn
    int n = -1, c = chunks;
    uint32_t set = 0;
    Weights<TYPE, 1> w;
    const auto move = [&](int by) {
        for (c += by; c >= chunks; c -= chunks, ++n) {
        }
        const uint16_t* at = d.down + (int64_t)__builtin_amdgcn_readlane(expert, n) * d.down_expert;
        set = (uint32_t)__builtin_amdgcn_readlane((int)members, n);
        w = {{at + row0 * d.down_stride, at + row1 * d.down_stride}};
    };
    const int mine = (units - wave + FEW_WAVES - 1) / FEW_WAVES;
    int asked = 0;
    auto load = [&](Unit& f, int i) {
        if (i >= asked) move(asked++ ? FEW_WAVES : wave);             // (past the end: the last one again)
        f.c = c, f.pair = nth(set);
        w.ask(f.w, c * 64, d.inter);
        const uint16_t* xp = d.acts + (int64_t)(f.pair < 0 ? (int)__builtin_ctz(set) : f.pair) * 2 * d.inter_pad + 8 * q + c * 64;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            f.x[s][0] = *reinterpret_cast<const uint4*>(xp + 32 * s);
            f.x[s][1] = *reinterpret_cast<const uint4*>(xp + d.inter_pad + 32 * s);
        }
    };
    auto multiply = [&](Unit& f, int) {
        if (f.c * 64 + 64 > d.inter) w.settle(f.w, f.c * 64, d.inter);
        w.stage(f.w, stage);
        const f4_t v = chunk_sum<TYPE>(w.fragment(stage, 0, 0), w.fragment(stage, 0, 1), f.x);
        if (f.pair >= 0) parts[(f.pair * chunks + f.c) * 4 + q] = v;
    };
    Unit f[U];
    pipeline(f, mine, load, multiply);
    __syncthreads();
    if (threadIdx.x < pairs * 4) {
        f4_t v = {0.f, 0.f, 0.f, 0.f};
        if (there[threadIdx.x >> 2])
            for (int i = 0; i < chunks; ++i) v += parts[((threadIdx.x >> 2) * chunks + i) * 4 + (threadIdx.x & 3)];
        sums[threadIdx.x] = v * HIGH<TYPE>;
    }
    __syncthreads();
    if (my_row < d.rows) {
        f4_t v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < d.slots; ++s) {
            const int pair = my_row * d.slots + s;
            const f4_t y = sums[pair * 4 + (threadIdx.x & 3)];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = there[pair] ? fmaf(weight[pair], y[j], v[j]) : v[j];
        }
        finish(d, my_row, my_col, v, residual);
    }
}
static_assert(FEW_PAIRS <= 16 && FEW_PAIRS * 4 <= 64 * FEW_WAVES, "one tile of members, a thread an output");

template <int TYPE, int EB, int RB>
hipError_t launch_up(hipStream_t s, const Experts16Job& d, int64_t leaders) {
    experts16_up_kernel<TYPE, EB, RB><<<dim3((unsigned)(leaders * (d.inter_pad / (8 * EB)))), 64 * UP_WAVES, 0, s>>>(d);
    return hipGetLastError();
}
template <int TYPE, int RB>
hipError_t launch(hipStream_t s, const Experts16Job& d) {
    const int64_t pairs = (int64_t)d.rows * d.slots, leaders = pairs < d.experts ? pairs : d.experts;
    const bool few = pairs <= FEW_PAIRS && pairs * (d.inter_pad / 64) <= FEW_UNITS && d.inter >= 8;
    hipError_t e;
    if constexpr (RB == 1)
        e = leaders * (d.inter_pad / 16) < 320 ? launch_up<TYPE, 1, 1>(s, d, leaders) : launch_up<TYPE, 2, 1>(s, d, leaders);
    else
        e = launch_up<TYPE, 2, RB>(s, d, leaders);
    if (e != hipSuccess) return e;
    if (few) {
        experts16_few_kernel<TYPE><<<dim3((unsigned)((d.hidden + 15) / 16)), 64 * FEW_WAVES, 0, s>>>(d);
        return hipGetLastError();
    }
    experts16_down_kernel<TYPE, RB>
        <<<dim3((unsigned)(leaders * ((d.hidden + DOWN_COLS - 1) / DOWN_COLS))), 64 * DOWN_WAVES, 0, s>>>(d);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    const int64_t threads = (int64_t)d.rows * (d.hidden_pad / 4);
    experts16_combine_kernel<<<dim3((unsigned)((threads + 255) / 256)), 256, 0, s>>>(d);
    return hipGetLastError();
}

int padded(int n, int to) { return (n + to - 1) / to * to; }

}  // namespace

size_t experts16_workspace(int rows, int slots, int hidden, int inter) {
    return (size_t)rows * slots * (4 * (size_t)padded(inter, 64) + 4 * (size_t)padded(hidden, 4));
}

hipError_t launch_experts16(hipStream_t s, Experts16Job d, void* workspace) {
    d.inter_pad = padded(d.inter, 64), d.hidden_pad = padded(d.hidden, 4);
    d.acts = static_cast<uint16_t*>(workspace);
    d.y = reinterpret_cast<float*>(d.acts + (size_t)d.rows * d.slots * 2 * d.inter_pad);
    const bool few = d.rows <= 16;                                    // (rows pick an expert once: one pass of 16)
    if (d.type == TYPE_BF16) return few ? launch<TYPE_BF16, 1>(s, d) : launch<TYPE_BF16, 4>(s, d);
    return few ? launch<TYPE_F16, 1>(s, d) : launch<TYPE_F16, 4>(s, d);
}

}  // namespace gfr
