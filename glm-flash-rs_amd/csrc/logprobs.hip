// Log probabilities of given tokens under rows of logits, the rows' entropies and their most likely tokens. With z = l / T,
// m = max z and S = sum of exp(z - m):
//   log p(t) = z_t - m - log S,   H = log S - (sum of (z - m) exp(z - m)) / S
// Masked logits (-inf, NaN) have probability 0; several of +inf share it equally.
//
// A row of up to 32768 logits is a workgroup's, a longer one is cut into chunks of one each, which a second launch joins. A
// chunk's logits stay in registers as they were loaded: their maximum first, then the sums against it, so that the row is read
// once and nothing is rescaled. S is held as C, the number of logits that equal the maximum, and R, the sum over the others:
// where one token has nearly all of the probability, log S = log(1 + R) keeps what 1 + R would round off.
// The most likely tokens of a chunk: maxima of sets of its logits give a threshold that as many logits reach as are asked
// for, and few more. These go to LDS, each counts those before it in the order (larger logits first, the lower token first
// among equal ones), and that is its place. Where more reach it than LDS has room for (rows of one value, a set far below the
// others), the places are filled one by one.
//
// Bound: HBM, the logits read once; next to it VALU issue, 15 instructions a logit, half of them a chunk's fixed part (4096 rows
// of 160000 bf16 with 4 places 264 us, 4960 GB/s; without places 232, 5640; fp32 2048 rows 212, 6180). The threshold and the
// places are what the difference is: a chain of two barriers and LDS for each of three workgroups a CU. Short calls are latency: 1 x 160000
// with 20 places 13 us (two launches), 16 x 131072 10.2, 77 x 32003 9.0, 1 x 4000 5.2.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lanes.hpp"
#include "launch.hpp"
#include "values.hpp"

namespace gfr {
namespace {


// A chunk's share of its row: the largest logit, how many equal it, the sums of the others' exponentials and of
// (l - largest) times these (logits before they are divided by the temperature).
struct Share {
    float most, count, rest, slope;
};

// A place in the order: larger logits first, the lower token first among equal ones, as integers (0: an empty place).
__device__ __forceinline__ uint64_t place_of(float logit, int token) {
    const uint32_t b = __builtin_bit_cast(uint32_t, logit + 0.f);     // (-0 is 0)
    return (uint64_t)(b ^ (b >> 31 ? 0xffffffffu : 0x80000000u)) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ int token_of(uint64_t place) { return (int)~(uint32_t)place; }
__device__ __forceinline__ float logit_of(uint64_t place) {
    const uint32_t b = (uint32_t)(place >> 32);
    return __builtin_bit_cast(float, b ^ (b >> 31 ? 0x80000000u : 0xffffffffu));
}

// Eight logits of a chunk from column c on, -inf from column end on.
template <int TYPE>
__device__ __forceinline__ Eight load_logits(const void* row, int64_t c, int64_t end) {
    if (c + 8 <= end) return load_some(row, TYPE, c, 8);
    constexpr uint32_t MASKED = TYPE == TYPE_BF16 ? 0xff80 : TYPE == TYPE_F16 ? 0xfc00 : 0xff800000;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        w[j] = MASKED;
        if (c + j < end) w[j] = TYPE == TYPE_F32 ? static_cast<const uint32_t*>(row)[c + j] : static_cast<const uint16_t*>(row)[c + j];
    }
    Eight e;
    if constexpr (TYPE == TYPE_F32) {
        e.a = make_uint4(w[0], w[1], w[2], w[3]), e.b = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
        e.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
        e.b = make_uint4(0, 0, 0, 0);
    }
    return e;
}

// The logits of a group, converted anew by instructions that the compiler takes for others each time: it would keep the
// values of one use for the next, in twice the registers.
template <int TYPE>
__device__ __forceinline__ f8_t fresh(const Eight& e) {
    if constexpr (TYPE == TYPE_F32) return values(e, TYPE);
    const uint32_t h[4] = {e.a.x, e.a.y, e.a.z, e.a.w};
    f8_t l;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float lo, hi;
        if constexpr (TYPE == TYPE_BF16)
            asm volatile("v_lshlrev_b32 %0, 16, %2\n\tv_and_b32 %1, 0xffff0000, %2" : "=&v"(lo), "=v"(hi) : "v"(h[j]));
        else
            asm volatile("v_cvt_f32_f16 %0, %2\n\tv_cvt_f32_f16_sdwa %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:WORD_1"
                         : "=&v"(lo), "=v"(hi) : "v"(h[j]));
        l[2 * j] = lo, l[2 * j + 1] = hi;
    }
    return l;
}

// A logit that at least `top` of a chunk's logits reach, and few more: one that the maxima of `top` to `top` + 3 of the chunk's 64
// sets reach, by halving (6 logits reach it for 4 places, 27 for 20, 55 for 32 on average; against the least of eight sets'
// maxima, and the place's largest of 64 by comparing each with each, 4096 rows of 160000 with 4 places 256 -> 247 us, with 32
// 330 -> 298, 3137 of 5888 fp16 with 20 34.1 -> 27.5). Where fewer sets hold a logit that is not masked, all that are not do;
// where halving ends early (equal maxima), more. Infinities and values far below the others are no bounds to halve between.
__device__ __forceinline__ float threshold(float set, float most, int top) {
    const bool any = set > -INFINITY;
    int reach = __popcll(__ballot(any));
    if (reach < top) return -3.402823466e38f;
    float lo = -max_over(64, any ? -set : -INFINITY), hi = most;
    if (hi == INFINITY) hi = max_over(64, set < INFINITY ? set : -INFINITY);
    if (hi - lo > 64.f) {
        const int n = __popcll(__ballot(set >= hi - 32.f));
        if (n >= top) lo = hi - 32.f, reach = n;
    }
    for (int i = 0; i < 16 && reach > top + 3; ++i) {
        const float mid = lo + 0.5f * (hi - lo);
        if (!(mid > lo && mid < hi)) break;
        const int n = __popcll(__ballot(set >= mid));
        if (n >= top) lo = mid, reach = n;
        else hi = mid;
    }
    return lo;
}

// A row's results from its sums: the entropy, the tokens' log probabilities (thread `from` of `threads` on), a place's.
struct Row {
    float most, log_sum;
    // (halves: the difference of two finite logits may pass the range where its quotient does not)
    __device__ __forceinline__ float log_p(const LogprobsJob& d, float l) const {
        if (!(l > -INFINITY)) return -INFINITY;
        return (l == most ? 0.f : 2.f * ((0.5f * l - 0.5f * most) / d.temperature)) - log_sum;
    }
    __device__ __forceinline__ void tokens(const LogprobsJob& d, int row, int from, int threads) const {
        for (int i = from; i < d.tokens; i += threads) {
            const int64_t at = (int64_t)row * d.tokens_stride + i;
            const int64_t token = d.wide_tokens ? static_cast<const int64_t*>(d.token)[at] : static_cast<const int32_t*>(d.token)[at];
            const bool there = token >= 0 && token < d.vocab;         // a token that is not in the vocabulary: probability 0
            d.logprob[(int64_t)row * d.tokens + i] =
                there ? log_p(d, load_one(d.logits, d.type, (int64_t)row * d.stride + token)) : -INFINITY;
        }
    }
    __device__ __forceinline__ void place(const LogprobsJob& d, int row, int i, uint64_t p) const {
        d.top_ids[(int64_t)row * d.top + i] = token_of(p);
        d.top_logprobs[(int64_t)row * d.top + i] = log_p(d, logit_of(p));
    }
    // Fewer logits than places are not masked: from place i on the masked tokens in order, enough of which are among the first
    // 64. One wave.
    __device__ __forceinline__ void masked(const LogprobsJob& d, int row, int i) const {
        const int lane = threadIdx.x & 63;
        const bool masked = lane < d.vocab && !(load_one(d.logits, d.type, (int64_t)row * d.stride + lane) > -INFINITY);
        const int at = i + set_before(__ballot(masked));
        if (!masked || at >= d.top) return;
        d.top_ids[(int64_t)row * d.top + at] = lane;
        d.top_logprobs[(int64_t)row * d.top + at] = -INFINITY;
    }
};
__device__ __forceinline__ Row row_of(const LogprobsJob& d, int row, const Share& s, bool writes) {
    const Row r = {s.most, logf(s.count) + log1pf(s.rest / s.count)};
    if (writes) d.entropy[row] = s.count > 0.f ? r.log_sum - s.slope / d.temperature / (s.count + s.rest) : 0.f;
    return r;
}

// V groups of eight logits a thread: group g of thread i starts at the chunk's column 8 (g THREADS + i).
// ONE: the chunk is its row, and there is no second launch.
template <int TYPE, int THREADS, int V, bool ONE>
__global__ void __launch_bounds__(THREADS) logprobs_chunk_kernel(LogprobsJob d) {
    constexpr int WAVES = THREADS / 64, ROOM = 2 * THREADS;
    __shared__ float maxima[WAVES][64];
    __shared__ float sums[WAVES][3];
    __shared__ uint64_t places[ROOM];
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = ONE ? (int)blockIdx.x : blockIdx.x / d.chunks, chunk = ONE ? 0 : blockIdx.x % d.chunks;
    const int64_t c0 = (int64_t)chunk * d.span, end = c0 + d.span < d.vocab ? c0 + d.span : d.vocab;
    const char* logits = static_cast<const char*>(d.logits) + (int64_t)row * d.stride * (TYPE == TYPE_F32 ? 4 : 2);
    Eight raw[V];
#pragma unroll
    for (int g = 0; g < V; ++g) raw[g] = load_logits<TYPE>(logits, c0 + 8 * (g * THREADS + tid), end);
    if (tid == 0) found = 0;
    float each[V], most = -INFINITY;                                  // (fmaxf leaves NaN out)
#pragma unroll
    for (int g = 0; g < V; ++g) {
        const f8_t l = fresh<TYPE>(raw[g]);
        each[g] = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) each[g] = fmaxf(each[g], l[j]);
        most = fmaxf(most, each[g]);
    }
    maxima[wave][lane] = most;
    __syncthreads();
    // each lane's maximum over the waves: 64 sets of logits whose columns lie among each other
    float set = maxima[0][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) set = fmaxf(set, maxima[w][lane]);
    const float M = max_over(64, set);
    const float least = d.top ? threshold(set, M, d.top) : 0.f;

    // exp(z) = exp2((l - M) by): the distance from the largest logit is taken first, one rounding of it, so that a term's error
    // goes by |z| and not by M. (A fused l by - M by, one instruction less, has the rounding of M by in every term: at M / T of
    // 1000 up to 4e-5 of it, and beyond 1e9 no small factor.) slope is summed in logits.
    const auto distance = [&](float l) { return fmaxf(l - M, -1e30f); };   // -1e30: masked (and NaN), exp2 of it is 0
    float rest = 0.f, slope = 0.f, count = 0.f;
#pragma unroll
    for (int g = 0; g < V; ++g) {
        // (two loops and no third that serves both: the compiler would merge them, and do the work of both for every group)
        if (__ballot(each[g] >= M)) {                                 // few: the maximum itself, and groups of masked ones
            const f8_t l = fresh<TYPE>(raw[g]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = distance(l[j]), e = __builtin_amdgcn_exp2f(x * d.by);
                if (l[j] == M) count += 1.f;
                else rest += e, slope = fmaf(x, e, slope);
            }
            asm volatile("; the maximum's group" : "+v"(rest), "+v"(slope), "+v"(count));
        } else {
            const f8_t l = fresh<TYPE>(raw[g]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = distance(l[j]), e = __builtin_amdgcn_exp2f(x * d.by);
                rest += e, slope = fmaf(x, e, slope);
            }
            asm volatile("; another group" : "+v"(rest), "+v"(slope));
        }
    }
    if (M == -INFINITY) count = rest = slope = 0.f;
    rest = sum_over(64, rest), slope = sum_over(64, slope), count = sum_over(64, count);
    if (lane == 0) sums[wave][0] = rest, sums[wave][1] = slope, sums[wave][2] = count;
    if (d.top && most >= least) {
#pragma unroll
        for (int g = 0; g < V; ++g)
            if (each[g] >= least) {
                const f8_t l = fresh<TYPE>(raw[g]);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (l[j] >= least) {
                        const int at = atomicAdd(&found, 1);
                        if (at < ROOM) places[at] = place_of(l[j], (int)(c0 + 8 * (g * THREADS + tid) + j));
                    }
            }
    }
    __syncthreads();
    // the sums in the first lanes of every wave of a row's only chunk, or of the first one
    Share s = {M, 0.f, 0.f, 0.f};
    if (ONE || tid < WAVES) {
        const int w = lane & (WAVES - 1);
        s.count = sum_over(WAVES, sums[w][2]), s.rest = sum_over(WAVES, sums[w][0]), s.slope = sum_over(WAVES, sums[w][1]);
    }
    Row r;
    uint64_t* out = nullptr;
    if constexpr (ONE) {
        r = row_of(d, row, s, tid == 0);
        r.tokens(d, row, THREADS - 1 - tid, THREADS);
    } else {
        const int64_t part = (int64_t)row * d.chunks + chunk;
        if (tid == 0) static_cast<Share*>(d.shares)[part] = s;
        out = static_cast<uint64_t*>(d.places) + part * d.top;
    }
    if (!d.top) return;
    const auto put = [&](int i, uint64_t p) {
        if constexpr (ONE) r.place(d, row, i, p);
        else out[i] = p;
    };
    const int n = found;
    if (n <= ROOM) {
        if constexpr (ONE) {
            if (wave == 0 && n < d.top) r.masked(d, row, n);
        } else {
            if (tid >= n && tid < d.top) out[tid] = 0;
        }
        // 2^by lanes count those before a place
        int by = 6;
        while (by && n << by > THREADS) --by;
        for (int i = tid >> by; i < n; i += THREADS >> by) {
            const uint64_t p = places[i];
            int before = 0;
            for (int o = tid & ((1 << by) - 1); o < n; o += 1 << by) before += places[o] > p;
            before = sum_over(1 << by, before);
            if (before < d.top && (tid & ((1 << by) - 1)) == 0) put(before, p);
        }
        return;
    }
    uint64_t last = ~0ull;
    for (int i = 0; i < d.top; ++i) {                                 // (more than ROOM: none of them stays empty)
        uint64_t best = 0;
#pragma unroll 1
        for (int g = 0; g < V; ++g) {                                 // (loaded again: registers hold no index)
            const int64_t c = c0 + 8 * (g * THREADS + tid);
            const f8_t l = values(load_logits<TYPE>(logits, c, end), TYPE);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint64_t p = place_of(l[j], (int)c + j);
                if (l[j] > -INFINITY && p < last && p > best) best = p;
            }
        }
        best = max_over(64, best);
        __syncthreads();
        if (lane == 0) places[wave] = best;
        __syncthreads();
        last = places[0];
        for (int w = 1; w < WAVES; ++w) last = larger(last, places[w]);
        if (tid == 0) put(i, last);
    }
}

// A workgroup a row: the chunks' shares against the row's largest logit, in every wave; the tokens in all waves, the places
// in the first.
constexpr int JOIN = 256;
__global__ void __launch_bounds__(JOIN) logprobs_join_kernel(LogprobsJob d) {
    extern __shared__ uint64_t places[];
    const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.x;
    const uint64_t* from = static_cast<const uint64_t*>(d.places) + (int64_t)row * d.chunks * d.top;
    for (int i = tid; i < d.chunks * d.top; i += JOIN) places[i] = from[i];
    Share s = {-INFINITY, 0.f, 0.f, 0.f};
    if (lane < d.chunks) s = static_cast<const Share*>(d.shares)[(int64_t)row * d.chunks + lane];
    const float M = max_over(64, s.most);
    float count = s.count, rest = s.rest, slope = s.slope;
    if (s.most < M) {
        const float x = fmaxf(s.most - M, -1e30f), e = __builtin_amdgcn_exp2f(x * d.by), all = s.count + s.rest;
        count = 0.f, rest = all * e, slope = e * fmaf(x, all, s.slope);
    }
    count = sum_over(64, count), rest = sum_over(64, rest), slope = sum_over(64, slope);
    const Row r = row_of(d, row, {M, count, rest, slope}, tid == 0);
    r.tokens(d, row, JOIN - 1 - tid, JOIN);                           // (from the last wave on: the first has the places)
    if (!d.top) return;
    // a chunk's places are in order, so that the next one is the largest of the chunks' heads
    __syncthreads();
    if (tid >= 64) return;
    const int end = lane < d.chunks ? (lane + 1) * d.top : 0;
    int next = lane * d.top;
    const auto take = [&] { return next < end ? places[next++] : 0; };
    uint64_t head = take(), after = take(), kept = 0;
    int i = 0;
    for (; i < d.top; ++i) {
        const uint64_t best = max_over(64, head);
        if (!best) break;
        if (lane == i) kept = best;
        if (head == best) head = after, after = take();
    }
    if (lane < i) r.place(d, row, lane, kept);
    if (i < d.top) r.masked(d, row, i);
}

// A row of at most 8 * 8 * 512 logits is one chunk, of the fewest groups that hold it: of 512 threads, or of 128 or 256 where
// there are rows for every CU, as long as 8 groups of a thread hold a row: more rows are under way at once, and barriers join
// fewer waves (us with 512 threads in two launches, in one, with fewer: 8192 rows of 1000 118, 47, 19; 8192 of 4000 without
// places -, 37, 18; 8192 of 8000 with 4 -, 57, 35; 4096 of 16000 with 32 -, 47, 41; 2000 of 8000 without -, 13.9, 11.2; one of
// 4000 11.6, 5.2, 7.0. 16 groups of 256 threads for longer rows: 8192 of 32000 97 -> 90, but 1200 of them with 20 25.0 -> 25.8).
constexpr int WIDE = 512, NARROW = 128, MOST = 8 * 8 * WIDE;

template <int TYPE, int THREADS, int V>
hipError_t launch_rows(hipStream_t s, const LogprobsJob& d) {
    logprobs_chunk_kernel<TYPE, THREADS, V, true><<<dim3((unsigned)d.rows), THREADS, 0, s>>>(d);
    return hipGetLastError();
}
template <int TYPE, int V>
hipError_t launch_chunks(hipStream_t s, const LogprobsJob& d) {
    logprobs_chunk_kernel<TYPE, WIDE, V, false><<<dim3((unsigned)(d.rows * (int64_t)d.chunks)), WIDE, 0, s>>>(d);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    logprobs_join_kernel<<<dim3((unsigned)d.rows), JOIN, (size_t)d.chunks * d.top * sizeof(uint64_t), s>>>(d);
    return hipGetLastError();
}
template <int TYPE>
hipError_t launch(hipStream_t s, const LogprobsJob& d, int groups) {
    if (d.chunks == 1) {
        if (d.rows >= 1024 && d.vocab <= 128 * NARROW) {
            if (d.vocab <= 8 * NARROW) return launch_rows<TYPE, NARROW, 1>(s, d);
            if (d.vocab <= 16 * NARROW) return launch_rows<TYPE, NARROW, 2>(s, d);
            if (d.vocab <= 32 * NARROW) return launch_rows<TYPE, NARROW, 4>(s, d);
            return d.vocab <= 64 * NARROW ? launch_rows<TYPE, NARROW, 8>(s, d) : launch_rows<TYPE, 2 * NARROW, 8>(s, d);
        }
        if (d.vocab <= 8 * WIDE) return launch_rows<TYPE, WIDE, 1>(s, d);
        if (d.vocab <= 16 * WIDE) return launch_rows<TYPE, WIDE, 2>(s, d);
        return d.vocab <= 32 * WIDE ? launch_rows<TYPE, WIDE, 4>(s, d) : launch_rows<TYPE, WIDE, 8>(s, d);
    }
    switch (groups) {
        case 1: return launch_chunks<TYPE, 1>(s, d);
        case 2: return launch_chunks<TYPE, 2>(s, d);
        case 4: return launch_chunks<TYPE, 4>(s, d);
        default: return launch_chunks<TYPE, 8>(s, d);
    }
}

// Groups of eight logits a thread of longer rows: 8, and fewer where that leaves CUs idle, as long as a row has no more
// chunks than the join has lanes. (4096 rows of 160000 bf16, top 4, with 2, 4 and 8 groups: 440, 304 and 264 us.)
int chunks_of(int vocab, int groups) { return (int)(((int64_t)vocab + 8 * WIDE * groups - 1) / (8 * WIDE * groups)); }
int groups_of(int rows, int vocab) {
    int v = 8;
    if (vocab <= MOST) return v;
    while (v > 1 && (int64_t)rows * chunks_of(vocab, v) < 512 && chunks_of(vocab, v / 2) <= 64) v /= 2;
    return v;
}

}  // namespace

int logprobs_chunks(int rows, int vocab) { return chunks_of(vocab, groups_of(rows, vocab)); }
size_t logprobs_workspace(int rows, int vocab, int top) {
    const int chunks = logprobs_chunks(rows, vocab);
    return chunks == 1 ? 0 : (size_t)rows * chunks * (sizeof(Share) + top * sizeof(uint64_t));
}

hipError_t launch_logprobs(hipStream_t s, LogprobsJob d, void* workspace) {
    const int groups = groups_of(d.rows, d.vocab);
    d.chunks = chunks_of(d.vocab, groups);
    d.span = ((d.vocab + d.chunks - 1) / d.chunks + 7) / 8 * 8;
    d.shares = workspace;
    d.places = static_cast<char*>(workspace) + (size_t)d.rows * d.chunks * sizeof(Share);
    if (d.type == TYPE_BF16) return launch<TYPE_BF16>(s, d, groups);
    return d.type == TYPE_F16 ? launch<TYPE_F16>(s, d, groups) : launch<TYPE_F32>(s, d, groups);
}

}  // namespace gfr
