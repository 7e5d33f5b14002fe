// The general router gate: logits -> picks and weights, for the gates that route.hpp's two do not cover (scores that are
// a softmax over all experts, kept as they are or renormalised; a bias for balance on either score; groups of experts of
// which only the best are chosen from; 16-bit logits, row strides; experts masked by -inf).
//
//   score[e]  = softmax over the live logits, or 1 / (1 + exp(-l[e]))
//   choice[e] = score[e] + bias[e]; without a bias the logit itself, which has the scores' order
//   groups    : E / G contiguous experts each; a group's value is its largest choice, or the sum of its two largest
//               (without a bias: of the two largest scores); the K groups of the largest values stay (equal: lower index)
//   picks     : the topk largest choices in the groups that stay, descending (equal: lower id)
//   weight    = score[pick], divided by (the picks' sum in slot order + 1e-20) if renormalised, times scale
// An expert whose logit or choice is -inf or NaN is masked: no group value counts it, the softmax leaves out its logit,
// and it is picked only where a row's kept groups have too few others, by lower id, with weight 0.
//
// 32768 rows of 256 (the first gate above) take 29 us, the bytes 7 of them at a copy's rate. Half of the 29 does not grow
// with the rows: a launch, one wave's chain of loads, sort and rounds, and behind it the 64-bit order of near choices (one
// wave of 27; one of 320 decides everything again). The other half, 13 to 14 us per 32768 rows, is about the issue of 316
// VALU instructions a row: a fifth the scores, a fifth the keys and their sort, a third the rounds. A third of the wave
// cycles wait. In 64-bit arithmetic throughout, a wave a row, they took 65 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "exl3_format.hpp"
#include "lanes.hpp"
#include "launch.hpp"

namespace gfr {
namespace {

__device__ __forceinline__ float logit_at(const void* l, int type, size_t i) {
    if (type == TYPE_F32) return static_cast<const float*>(l)[i];
    const uint16_t h = static_cast<const uint16_t*>(l)[i];
    return type == TYPE_BF16 ? __builtin_bit_cast(float, (uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}

// ---- a row's lanes --------------------------------------------------------------------------------------------------
// W neighbouring lanes hold a row, 64 / W rows a wave. They are dealt to the groups (the power of two at or above G of
// them, lpg lanes each); a lane holds up to PER consecutive experts of its group, so that experts ascend with (lane,
// register) and the lowest lane among equals has the lowest id.
template <int W>
struct RowLanes {
    int lane, t, first;                                            // lane of the wave, of the row, the row's first lane
    __device__ __forceinline__ RowLanes() : lane(threadIdx.x & 63), t(lane % W), first(lane - t) {}
    // the lowest lane of the row whose bit is set in a ballot
    __device__ __forceinline__ int lowest(uint64_t ballot) const {
        if constexpr (W == 64) return __builtin_ctzll(ballot);
        const uint32_t half = lane & 32 ? (uint32_t)(ballot >> 32) : (uint32_t)ballot;
        if constexpr (W == 32) return first + __builtin_ctz(half | 0x80000000u);
        return first + __builtin_ctz((half >> (lane & 16)) | 0x8000u);
    }
};

template <int W, typename T>
__device__ __forceinline__ T row_max(T v) { return max_over(W, v); }
template <int W, typename T>
__device__ __forceinline__ T row_sum(T v) { return sum_over(W, v); }

// Which groups stay: the row's group values, one in all lanes of a group. gap: how far the last that stays is above the
// first that does not (NaN where both are infinite).
template <int W, typename T>
__device__ __forceinline__ bool group_stays(const GateJob& g, const RowLanes<W>& r, int group, T value, T& gap) {
    int before = 0;
    for (int q = 0; q < g.groups; ++q) {
        const T other = __shfl(value, r.first + q * g.lpg);
        before += other > value || (other == value && q < group);
    }
    const bool in = group < g.groups, stays = in && before < g.kept;
    const T low = -row_max<W>(stays ? -value : (T)-__builtin_inf()), high = row_max<W>(in && !stays ? value : (T)-__builtin_inf());
    gap = low - high;
    return stays;
}

// n consecutive values (0 <= n <= PER) from p[at] on; those past n are -inf. four: groups of four are aligned and whole.
// Every load is issued, those past the end at the last value's place, so that none waits for another. (A lane without
// values reads p[at], which the caller makes a valid place.)
template <int PER>
__device__ __forceinline__ void load_values(const void* p, int type, size_t at, int n, bool four, float (&v)[PER]) {
    const int last = n > 0 ? n - 1 : 0;
    const float* f = static_cast<const float*>(p) + at;
    const uint16_t* h = static_cast<const uint16_t*>(p) + at;
    if (PER >= 4 && four) {
        const int quad = last & ~3;
        if (type == TYPE_F32) {
#pragma unroll
            for (int j = 0; j + 3 < PER; j += 4) {
                const float4 q = *reinterpret_cast<const float4*>(f + min(j, quad));
                v[j] = q.x, v[j + 1] = q.y, v[j + 2] = q.z, v[j + 3] = q.w;
            }
        } else {
            ushort4 q[PER / 4 ? PER / 4 : 1];
#pragma unroll
            for (int j = 0; j + 3 < PER; j += 4) q[j / 4] = *reinterpret_cast<const ushort4*>(h + min(j, quad));
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const uint16_t e = j % 4 == 0 ? q[j / 4].x : j % 4 == 1 ? q[j / 4].y : j % 4 == 2 ? q[j / 4].z : q[j / 4].w;
                v[j] = type == TYPE_BF16 ? __builtin_bit_cast(float, (uint32_t)e << 16) : (float)__builtin_bit_cast(_Float16, e);
            }
        }
    } else if (type == TYPE_F32) {
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = f[min(j, last)];
    } else {
        uint16_t e[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) e[j] = h[min(j, last)];
#pragma unroll
        for (int j = 0; j < PER; ++j)
            v[j] = type == TYPE_BF16 ? __builtin_bit_cast(float, (uint32_t)e[j] << 16) : (float)__builtin_bit_cast(_Float16, e[j]);
    }
    if (n < PER) {
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = j < n ? v[j] : -__builtin_inff();
    }
}

// The row's picks as 64-bit arithmetic orders them: lane s of the row gets the s-th.
template <int W, int PER>
__device__ __forceinline__ void pick_exactly(const GateJob& g, size_t row_at, int n, int group, int base, int& pick,
                                             bool& live) {
    constexpr double NONE = -__builtin_inf();
    const RowLanes<W> r;
    float l[PER];
    load_values<PER>(g.logits, g.type, row_at + base, n, false, l);
    uint32_t have = n >= 32 ? 0xffffffffu : (1u << n) - 1u;        // this lane's experts that can still be picked
    double v[PER], top = NONE, total = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        v[j] = l[j] > -__builtin_inff() ? (double)l[j] : NONE;     // NaN: masked
        top = larger(top, v[j]);
    }
    top = row_max<W>(top);
    const bool scores = g.bias || (g.kept < g.groups && g.top2);
    if (scores && g.softmax) {
#pragma unroll
        for (int j = 0; j < PER; ++j) total += v[j] == NONE ? 0. : v[j] == top ? 1. : exp(v[j] - top);
        total = row_sum<W>(total);
    }
    const auto score = [&](double x) {
        if (g.softmax) return x == NONE ? 0. : (x == top ? 1. : exp(x - top)) / total;
        return 1. / (1. + exp(-x));
    };
    if (g.bias) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const double c = j < n && v[j] > NONE ? score(v[j]) + (double)g.bias[base + j] : NONE;
            v[j] = c > NONE ? c : NONE;
        }
    }
    if (g.kept < g.groups) {
        double a = NONE, b = NONE;                                 // the two largest
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            b = v[j] > a ? a : larger(b, v[j]);
            a = larger(a, v[j]);
        }
        stages_up_to<2>(g.lpg, [&](auto st) {
            const double pa = partner_of<decltype(st)::value>(a), pb = partner_of<decltype(st)::value>(b);
            b = a > pa ? larger(pa, b) : larger(a, pb);
            a = larger(a, pa);
        });
        if (g.top2) {
            if (!g.bias) a = a > NONE ? score(a) : NONE, b = b > NONE ? score(b) : NONE;
            if (b > NONE) a += b;
        }
        double gap;
        if (!group_stays<W>(g, r, group, a, gap)) {
            have = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = NONE;
        }
    }
    // topk rounds: the largest choice, of the lowest lane and register that hold it; where none is left, the lowest
    // masked expert
    for (int s = 0; s < g.topk; ++s) {
        double mine = v[0];
#pragma unroll
        for (int j = 1; j < PER; ++j) mine = larger(mine, v[j]);
        const double best = row_max<W>(mine);
        const bool some = best > NONE;
        const uint64_t with = __ballot(mine == best), left = __ballot(have != 0);
        const int w = r.lowest(some ? with : left);
        int at = __builtin_ctz(have | 0x80000000u);
        if (some) {
            at = 0;
#pragma unroll
            for (int j = PER - 1; j >= 0; --j) at = v[j] == best ? j : at;
        }
        const int e = __shfl(base + at, w);
        if (r.lane == w) {
            have &= ~(1u << at);
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = j == at ? NONE : v[j];
        }
        if (r.t == s) {
            pick = e;
            live = some;
        }
    }
}

// ---- the picks in 32 bits -------------------------------------------------------------------------------------------
// A lane sorts its choices once, as integers of the floats' order whose low bits are replaced by 15 - register, so that a
// comparator is a max and a min; a round takes the largest of the lanes' heads, and its lane shifts by one. The order
// found is certain where neighbours in it (the picks, the first that is not picked, the last group that stays and the
// first that does not) differ by more than their errors: the 16 units in the last place that the low bits hide, and the
// scores' own. Where it is not, and for equal choices, the picks and those after them that may belong before one are put
// in order by their choices in 64 bits, one a lane; a wave with a row whose groups are in doubt, or with too few experts
// that are not masked, goes to pick_exactly. With 16-bit logits and no bias the choices are the logits, whose low ten
// bits are zero: the expert's place in the row stands there, and every order is certain.
constexpr int MASKED = (int)0x80000100, ABSENT = (int)0x80000000;
__device__ __forceinline__ int ordered(float v) {
    const int b = __builtin_bit_cast(int, v);
    return b ^ (int)((uint32_t)(b >> 31) >> 1);
}
// (low: the bits that hold a place. A negative 16-bit logit's are ones.)
__device__ __forceinline__ float unordered(int k, int low) {
    k &= ~low;
    if (low == 1023 && k < 0) k |= low;
    return __builtin_bit_cast(float, k ^ (int)((uint32_t)(k >> 31) >> 1));
}

template <int N>
__device__ __forceinline__ void sort_down(int (&k)[N]) {           // Batcher's odd-even merge sort
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int s = p; s >= 1; s /= 2)
#pragma unroll
            for (int j = s % p; j + s < N; j += 2 * s)
#pragma unroll
                for (int i = 0; i < s; ++i)
                    if (i + j + s < N && (i + j) / (2 * p) == (i + j + s) / (2 * p)) {
                        const int hi = max(k[i + j], k[i + j + s]), lo = min(k[i + j], k[i + j + s]);
                        k[i + j] = hi;
                        k[i + j + s] = lo;
                    }
}

template <int W, int PER>
__device__ __forceinline__ bool pick_fast(const GateJob& g, const RowLanes<W>& r, const float (&l)[PER], float (&part)[PER],
                                          const float (&bias)[PER], float top, float inverse, size_t row_at, int n, int group,
                                          int base, int* picked, int& pick, bool& live) {
    constexpr float NONE = -__builtin_inff(), LOG2E = 1.44269504088896341f;
    // keys
    const bool exact = !g.bias && g.type != TYPE_F32;              // every order is certain
    int k[PER];
    const int low = exact ? 1023 : 15;
    if (g.bias) {
#pragma unroll
        for (int j = 0; j < PER; ++j) part[j] = part[j] * inverse + bias[j];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const float c = g.bias ? part[j] : l[j] + 0.f;              // (+ 0: one zero)
        const int order = exact ? 1023 - (r.t * PER + j) : 15 - (j & 15);
        const bool is = l[j] > NONE && c > NONE;
        k[j] = is ? (ordered(c) & ~low) | order : (j < n ? MASKED : ABSENT) + (15 - (j & 15));
    }
    sort_down<PER>(k);

    // The error of a choice, in units of 2^-24. A score is off by at most 48 of the row's largest (softmax) or 8 (sigmoid):
    //   softmax: an exponential's argument l - top = -d takes three roundings and its value two units, 3 d + 2 of itself,
    //   at most 3.1 of the largest (d exp(-d) < 0.37); the sum of up to 1024 of them the exponentials' own, 3 x 4.4 + 2
    //   (the mean d, weighted with exp(-d), is below 4.4), and 22 additions of positive terms (16 in a lane, 6 over the
    //   lanes); the reciprocal and two products 4; sigmoid: s (1 - s) (3 |l| + 2) + 4 < 6.
    // The choice adds its sum's rounding and the 15 units in the last place that the low bits hide: 31 of itself, at
    // most 36 of its neighbour. Two such errors meet, and twice that is taken.
    constexpr float UNIT = 0x1p-24f;
    const float score_error = g.bias ? (g.softmax ? 48.f * inverse : 8.f) * UNIT : 0.f;
    const auto doubt = [&](float x) { return exact ? -1.f : 4.f * (score_error + 36.f * UNIT * fabsf(x)); };
    bool all_certain = true, order_certain = true;                 // false: pick_exactly; the candidates' order, below
    if (g.kept < g.groups) {
        int a = k[0], b = PER > 1 ? k[PER > 1 ? 1 : 0] : ABSENT;
        stages_up_to<2>(g.lpg, [&](auto st) {
            const int pa = (int)partner<decltype(st)::value>((uint32_t)a), pb = (int)partner<decltype(st)::value>((uint32_t)b);
            b = max(min(a, pa), max(b, pb));
            a = max(a, pa);
        });
        const bool has = a > MASKED + 15, two = b > MASKED + 15;
        float va = unordered(a, low), vb = unordered(b, low), value = has ? va : NONE, error = doubt(va);
        if (g.top2) {
            if (!g.bias) {
                const auto score = [&](float x) {
                    if (g.softmax) return (x == top ? 1.f : __builtin_amdgcn_exp2f((x - top) * LOG2E)) * inverse;
                    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -LOG2E));
                };
                // of two scores a group, two groups: a key's hidden bits (30 units of the logit) move a score by its slope
                // (at most the score, a sigmoid's a quarter) times them
                error = 4.f * UNIT * (g.softmax ? (48.f + 36.f * fmaxf(fabsf(va), fabsf(vb))) * inverse
                                                : 8.f + 9.f * fmaxf(fabsf(va), fabsf(vb)));
                va = score(va), vb = score(vb);
                value = has ? va : NONE;
            } else {
                error += two ? doubt(vb) : 0.f;
            }
            if (two) value = va + vb;
        }
        float gap;
        const bool stays = group_stays<W>(g, r, group, value, gap);
        error = row_max<W>(has ? error : 0.f);
        all_certain = (exact && !g.top2) || gap > error;
        if (!stays) {
#pragma unroll
            for (int j = 0; j < PER; ++j) k[j] = ABSENT;
        }
    }

    // Rounds: lane s gets the s-th key and its expert, through LDS, from the lane that held it. One more than the picks,
    // then more for as long as the next one may belong before a row's last pick.
    int key = ABSENT, found = 0;
    const auto rounds = [&](auto depth, int until) {
        constexpr int D = decltype(depth)::value;
        for (; found < until; ++found) {
            const int best = row_max<W>(k[0]);
            bool mine = k[0] == best;
            const uint64_t with = __ballot(mine);
            if (__builtin_popcountll(with) != 64 / W) {            // equal keys: the lowest lane's first
                mine = r.lane == r.lowest(with);
                order_certain = false;
            }
            if (mine) {
                picked[r.first + found] = base + (exact ? (1023 - (best & 1023)) % PER : 15 - (best & 15));
#pragma unroll
                for (int i = 0; i < D; ++i) k[i] = i + 1 < PER ? k[i + 1 < PER ? i + 1 : i] : ABSENT;
                if (D < PER && k[0] == best) all_certain = false;  // a lane of more than D pops has lost its order
            }
            key = r.t == found ? best : key;
        }
    };
    const auto more = [&](int until) {
        if (PER > 8 && g.topk <= 8) rounds(std::integral_constant<int, PER < 8 ? PER : 8>{}, until);
        else rounds(std::integral_constant<int, PER>{}, until);
    };
    more(g.topk + 1);
    const float v = unordered(key, low), behind = unordered(__shfl_down(key, 1), low);
    const bool here = key > MASKED + 15, next = r.t + 1 < W && __shfl_down(key, 1) > MASKED + 15;
    const bool near = r.t < g.topk && here && next && !(v - behind > doubt(v));
    if (r.t < g.topk && !here) all_certain = false;                // masked picks
    if (__any(near)) {
        order_certain = false;
        const float last = __shfl(v, r.first + g.topk - 1);
        while (__any(r.t == found - 1 && key > MASKED + 15 && !(last - unordered(key, low) > doubt(last)))) {
            if (found == W) {
                all_certain = false;
                break;
            }
            more(found + 1);
        }
    }
    __builtin_amdgcn_wave_barrier();
    pick = picked[r.lane];
    live = r.t < found && key > MASKED + 15;

    // Rows in doubt: the candidates' choices in 64 bits, each lane's place among them
    if (__any(!order_certain)) {
        double total = 0.;
        if (g.bias && g.softmax) {
            float l[PER];
            load_values<PER>(g.logits, g.type, row_at + base, n, g.four, l);
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (l[j] > NONE) total += l[j] == top ? 1. : exp((double)l[j] - (double)top);
            total = row_sum<W>(total);
        }
        double c = -__builtin_inf();
        if (live) {
            const float x = logit_at(g.logits, g.type, row_at + pick);
            c = x;
            if (g.bias) {
                c = g.softmax ? (x == top ? 1. : exp((double)x - (double)top)) / total : 1. / (1. + exp(-(double)x));
                c += (double)g.bias[pick];
            }
        }
        int place = live ? 0 : r.t;
        for (int q = 0; q < found; ++q) {
            const double other = __shfl(c, r.first + q);
            const int e = __shfl(pick, r.first + q);
            if (live) place += other > c || (other == c && e < pick);
        }
        pick = __builtin_amdgcn_ds_permute((r.first + place) * 4, pick);
    }
    live = live && r.t < g.topk;
    return all_certain;
}

template <int W, int PER, int THREADS>
__global__ void __launch_bounds__(THREADS) gate_kernel(GateJob g) {
    constexpr float NONE = -__builtin_inff();
    __shared__ int picked[THREADS];
    const RowLanes<W> r;
    const int64_t row = (int64_t)blockIdx.x * (THREADS / W) + threadIdx.x / W;
    const bool real = row < g.rows;
    const size_t at = (size_t)(real ? row : g.rows - 1) * g.stride;
    const int group = r.t / g.lpg, first = (r.t % g.lpg) * g.per_lane, at_expert = group * g.per_group + first;
    int n = g.per_group - first;                                   // experts of this lane: base .. base + n - 1
    n = group < g.groups && n > 0 ? (n < g.per_lane ? n : g.per_lane) : 0;
    const int base = n > 0 ? at_expert : 0;

    // logits (absent and masked ones -inf), the row's largest, the softmax's sum
    constexpr float LOG2E = 1.44269504088896341f;
    float top = NONE, total = 1.f;
    int pick = 0;
    bool live = false, certain = PER <= 16;                        // more a lane: few groups of many experts, exactly at once
    {
        float l[PER];
        float bias[PER];
        load_values<PER>(g.logits, g.type, at + base, n, g.four, l);
        if (g.bias) load_values<PER>(g.bias, TYPE_F32, base, n, g.four_bias, bias);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            l[j] = fmaxf(l[j], NONE);                              // NaN: masked
            top = fmaxf(top, l[j]);
        }
        float part[PER];                                           // exp(l - top), or the sigmoid
        if (g.softmax) {
            top = row_max<W>(top);
            total = 0.f;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                part[j] = l[j] == top ? 1.f : __builtin_amdgcn_exp2f((l[j] - top) * LOG2E);
                part[j] = l[j] > NONE ? part[j] : 0.f;
                total += part[j];
            }
            total = row_sum<W>(total);
        } else if (g.bias) {
#pragma unroll
            for (int j = 0; j < PER; ++j) part[j] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(l[j] * -LOG2E));
        }
        if constexpr (PER <= 16)
            certain = pick_fast<W, PER>(g, r, l, part, bias, top, g.softmax ? __builtin_amdgcn_rcpf(total) : 1.f, at, n, group,
                                        base, picked + (threadIdx.x & ~63), pick, live);
    }
    if (__any(!certain && real)) pick_exactly<W, PER>(g, at, n, group, base, pick, live);

    // the picks' weights
    float sc = 0.f;
    if (r.t < g.topk && live) {
        const float x = logit_at(g.logits, g.type, at + pick);
        sc = g.softmax ? (x == top ? 1.f : expf(x - top)) / total : 1.f / (1.f + expf(-x));
    }
    float weight = sc;
    if (g.renorm) {
        float sum = 0.f;
        for (int s = 0; s < g.topk; ++s) sum += __shfl(sc, r.first + s);
        weight = sc / (sum + 1e-20f);
    }
    weight *= g.scale;
    if (real && r.t < g.slots) {
        g.picks[row * g.slots + r.t] = r.t < g.topk ? pick : g.routed;
        g.weights[row * g.slots + r.t] = r.t < g.topk ? weight : 1.f;
    }
}

}  // namespace

template <int W, int THREADS>
static hipError_t launch_rows(hipStream_t s, const GateJob& g) {
    constexpr int ROWS = THREADS / W;
    const dim3 grid((unsigned)((g.rows + ROWS - 1) / ROWS));
    if (g.per_lane <= 1) gate_kernel<W, 1, THREADS><<<grid, THREADS, 0, s>>>(g);
    else if (g.per_lane <= 2) gate_kernel<W, 2, THREADS><<<grid, THREADS, 0, s>>>(g);
    else if (g.per_lane <= 4) gate_kernel<W, 4, THREADS><<<grid, THREADS, 0, s>>>(g);
    else if (g.per_lane <= 8) gate_kernel<W, 8, THREADS><<<grid, THREADS, 0, s>>>(g);
    else if (W < 64 || g.per_lane <= 16) gate_kernel<W, 16, THREADS><<<grid, THREADS, 0, s>>>(g);
    else gate_kernel<W, W == 64 ? 32 : 16, THREADS><<<grid, THREADS, 0, s>>>(g);
    return hipGetLastError();
}

hipError_t launch_gate(hipStream_t s, GateJob g) {
    int lanes = 1;
    while (lanes < g.groups) lanes *= 2;
    g.per_group = g.routed / g.groups;
    const auto deal = [&](int w) {
        g.lpg = w / lanes;
        g.per_lane = g.lpg ? (g.per_group + g.lpg - 1) / g.lpg : 64;
        return lanes <= w && g.topk < w && g.slots <= w && g.per_lane <= 16;
    };
    const auto four = [](const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (4 * bytes) == 0; };
    // Few rows: a wave a row, the shortest way through one. Many: as many rows a wave as hold their choices in 16
    // registers a lane. us at 64 / 32 / 16 lanes a row (fp32 logits; top-8 of 256, 4 of 8 groups, sigmoid and bias):
    //   4096 rows 12.8 / 13.4 / 17.2, 8192 15.6 / 15.4 / 18.3, 16384 24.2 / 19.7 / 21.1, 131072 134 / 86.8 / 68.8;
    // top-4 of 64, softmax and bias: 2048 rows 5.2 / 5.1 / 5.3, 4096 6.7 / 5.7 / 5.7, 32768 20.3 / 13.1 / 8.8; top-6 of
    // 160, 3 of 8 groups, bf16: 8192 rows 12.2 / 8.9 / 8.0, 32768 35.4 / 23.2 / 17.5
    int w = 64;
    for (int fewer = 16; fewer < 64 && w == 64; fewer *= 2)
        if (deal(fewer) && g.rows >= (g.per_lane <= 8 ? 4096 : 8192)) w = fewer;
    deal(w);
    const bool whole = g.per_lane % 4 == 0 && g.per_group % 4 == 0;
    g.four = whole && g.stride % 4 == 0 && four(g.logits, g.type == TYPE_F32 ? 4 : 2);
    g.four_bias = whole && four(g.bias, 4);
    if (w == 16) return launch_rows<16, 256>(s, g);
    if (w == 32) return launch_rows<32, 256>(s, g);
    return launch_rows<64, 64>(s, g);
}

}  // namespace gfr
