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
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "exl3_format.hpp"
#include "launch.hpp"

namespace gfr {
namespace {

// ---- reductions over the 2, 4 .. 64 lanes that share a value ---------------------------------------------------------
// Stage by stage each lane meets a lane of the other half of its next larger block (quad swaps, half-row and row
// mirrors, the permlane swaps), so that after the stages up to width w every lane of an aligned block of w has the
// block's result.
template <int STAGE>
__device__ __forceinline__ uint32_t partner(uint32_t v) {
    if constexpr (STAGE == 2) return lane_xor<1>(v);
    else if constexpr (STAGE == 4) return lane_xor<2>(v);
    else if constexpr (STAGE == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, false);   // row_half_mirror
    else if constexpr (STAGE == 16) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, false);  // row_mirror
    else if constexpr (STAGE == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (uint32_t)((__lane_id() & 16) ? r[0] : r[1]);
    } else {
        return lane_xor<32>(v);
    }
}
template <int STAGE, typename T>
__device__ __forceinline__ T partner_of(T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, partner<STAGE>(__builtin_bit_cast(uint32_t, v)));
    } else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, (uint64_t)partner<STAGE>((uint32_t)b) | (uint64_t)partner<STAGE>((uint32_t)(b >> 32)) << 32);
    }
}
template <int STAGE, typename F>
__device__ __forceinline__ void stages_up_to(int width, F f) {
    if constexpr (STAGE <= 64) {
        if (width >= STAGE) f(std::integral_constant<int, STAGE>{});
        stages_up_to<2 * STAGE>(width, f);
    }
}
template <typename T>
__device__ __forceinline__ T larger(T a, T b) { return a > b ? a : b; }
template <typename T>
__device__ __forceinline__ T max_over(int width, T v) {
    stages_up_to<2>(width, [&](auto s) { v = larger(v, partner_of<decltype(s)::value>(v)); });
    return v;
}
template <typename T>
__device__ __forceinline__ T sum_over(int width, T v) {
    stages_up_to<2>(width, [&](auto s) { v += partner_of<decltype(s)::value>(v); });
    return v;
}

__device__ __forceinline__ float logit_at(const void* l, int type, size_t i) {
    if (type == TYPE_F32) return static_cast<const float*>(l)[i];
    const uint16_t h = static_cast<const uint16_t*>(l)[i];
    return type == TYPE_BF16 ? __builtin_bit_cast(float, (uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}

// A wave routes one row. Its lanes are dealt to the groups (lanes = the power of two at or above G, LPG lanes a group);
// a lane holds C consecutive experts of its group, so that experts ascend with (lane, register) and the lowest lane among
// equals has the lowest id.
template <int PER>
__global__ void __launch_bounds__(64) gate_kernel(GateJob g) {
    using T = double;
    constexpr T NONE = -__builtin_inf();
    const int lane = threadIdx.x & 63;
    const int64_t row = blockIdx.x;
    const int group = lane / g.lpg, first = (lane % g.lpg) * g.per_lane, base = group * g.per_group + first;
    int n = g.per_group - first;                                   // experts of this lane: base .. base + n - 1
    n = group < g.groups && n > 0 ? (n < g.per_lane ? n : g.per_lane) : 0;
    const size_t at = (size_t)row * g.stride + base;

    // scores and choices
    T score[PER], v[PER];
    uint32_t have = n >= 32 ? 0xffffffffu : (1u << n) - 1u;        // this lane's experts that can still be picked
    T top = NONE, total = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        T l = NONE;
        if (j < n) l = (T)logit_at(g.logits, g.type, at + j);
        if (!(l > NONE)) l = NONE;                                 // NaN: masked
        v[j] = l;
        top = larger(top, l);
    }
    if (g.softmax) {
        top = max_over(64, top);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            score[j] = v[j] == NONE ? 0. : v[j] == top ? 1. : exp(v[j] - top);
            total += score[j];
        }
        total = sum_over(64, total);
#pragma unroll
        for (int j = 0; j < PER; ++j) score[j] = v[j] == NONE ? 0. : score[j] / total;
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) score[j] = 1. / (1. + exp(-v[j]));
    }
    if (g.bias) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            T c = NONE;
            if (j < n && v[j] > NONE) c = score[j] + (T)g.bias[base + j];
            v[j] = c > NONE ? c : NONE;
        }
    }

    // the groups that stay
    if (g.kept < g.groups) {
        T a = NONE, b = NONE;                                      // the two largest
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const T s = g.top2 && !g.bias ? (v[j] > NONE ? score[j] : NONE) : v[j];
            b = s > a ? a : larger(b, s);
            a = larger(a, s);
        }
        stages_up_to<2>(g.lpg, [&](auto st) {
            const T pa = partner_of<decltype(st)::value>(a), pb = partner_of<decltype(st)::value>(b);
            b = a > pa ? larger(pa, b) : larger(a, pb);
            a = larger(a, pa);
        });
        const T value = g.top2 && b > NONE ? a + b : a;
        int before = 0;
        for (int q = 0; q < g.groups; ++q) {
            const T other = __shfl(value, q * g.lpg);
            before += other > value || (other == value && q < group);
        }
        if (before >= g.kept) {
            have = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = NONE;
        }
    }

    // topk rounds: the largest choice, of the lowest lane and register that hold it
    int pick = 0;
    bool live = false;
    for (int s = 0; s < g.topk; ++s) {
        T mine = v[0];
#pragma unroll
        for (int j = 1; j < PER; ++j) mine = larger(mine, v[j]);
        const T best = max_over(64, mine);
        const bool some = best > NONE;
        const uint64_t m = some ? __ballot(mine == best) : __ballot(have != 0);
        const int w = __builtin_ctzll(m);
        int at_j = __builtin_ctz(have | 0x80000000u);              // none live: the lane's first that is left
        if (some) {
            at_j = 0;
#pragma unroll
            for (int j = PER - 1; j >= 0; --j) at_j = v[j] == best ? j : at_j;
        }
        const int e = __shfl(base + at_j, w);
        if (lane == w) {
            have &= ~(1u << at_j);
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = j == at_j ? NONE : v[j];
        }
        if (lane == s) {
            pick = e;
            live = some;
        }
    }

    // the picks' weights, in 32 bits from here on
    double sc = 0.;
    if (lane < g.topk && live) {
        const T l = (T)logit_at(g.logits, g.type, (size_t)row * g.stride + pick);
        sc = g.softmax ? (l == top ? 1. : exp(l - top)) / total : 1. / (1. + exp(-l));
    }
    double weight = sc;
    if (g.renorm) {
        double sum = 0.;
        for (int s = 0; s < g.topk; ++s) sum += __shfl(sc, s);
        weight = sc / (sum + 1e-20);
    }
    weight *= g.scale;
    if (lane < g.slots) {
        g.picks[row * g.slots + lane] = lane < g.topk ? pick : g.routed;
        g.weights[row * g.slots + lane] = lane < g.topk ? (float)weight : 1.f;
    }
}

}  // namespace

hipError_t launch_gate(hipStream_t s, GateJob g) {
    int lanes = 1;
    while (lanes < g.groups) lanes *= 2;
    g.lpg = 64 / lanes;
    g.per_group = g.routed / g.groups;
    g.per_lane = (g.per_group + g.lpg - 1) / g.lpg;
    const dim3 grid(g.rows);
    if (g.per_lane <= 1) gate_kernel<1><<<grid, 64, 0, s>>>(g);
    else if (g.per_lane <= 2) gate_kernel<2><<<grid, 64, 0, s>>>(g);
    else if (g.per_lane <= 4) gate_kernel<4><<<grid, 64, 0, s>>>(g);
    else if (g.per_lane <= 8) gate_kernel<8><<<grid, 64, 0, s>>>(g);
    else if (g.per_lane <= 16) gate_kernel<16><<<grid, 64, 0, s>>>(g);
    else gate_kernel<32><<<grid, 64, 0, s>>>(g);
    return hipGetLastError();
}

}  // namespace gfr
