// Direct-to-LDS loads and the waits around them, for kernels that stage their operands several steps ahead.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gfr {

// 16-byte direct-to-LDS load in the scalar-base form: lane i reads sbase + voff_i (32-bit unsigned per-lane offset) and
// its 16 bytes land at m0 + 16 i, so a per-step advance is one 64-bit scalar add and the LDS destination stays in
// scalar registers. Only the lanes of `mask` (uniform) load; the others' 16 bytes of LDS keep what they hold. An empty
// mask still counts as one load (vmcnt), so every wave's count a step is the same whatever it has to load. Called with
// all lanes active. Written as inline asm: the compiler treats its builtin as an LDS store of unknown address and puts
// s_waitcnt vmcnt(0) before every later LDS read, which drains the whole load pipeline each step; here the kernels wait
// for their stages themselves (wait_vmcnt), and loads complete in order, so any wait the compiler adds for its own loads
// only waits longer. The base goes through vcc by a scalar move: a VMEM instruction may read an SGPR that a VALU
// instruction wrote (the v_readlane of a spilled base, a v_readfirstlane) only five wait states later, and the compiler,
// which does not look into the asm, keeps no such distance; scalar instructions wait for VALU writes by themselves.
__device__ __forceinline__ void load_lds16_s(uint64_t sbase, uint32_t voff, uint32_t m0, uint64_t mask) {
    __asm__ volatile("s_mov_b64 exec, %3\n\ts_mov_b64 vcc, %1\n\tglobal_load_lds_dwordx4 %0, vcc\n\ts_mov_b64 exec, -1"
                     :: "v"(voff), "s"(sbase), "{m0}"(m0), "s"(mask) : "memory", "vcc");
}
// The LDS address (m0's unit) of shared memory.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    // readfirstlane returns int: through uint32_t, so that the low word is not sign-extended into the high one
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (uint64_t)lo | ((uint64_t)hi << 32);
}

// Workgroup barrier for LDS-only hand-offs: this wave's LDS operations complete, then s_barrier. Unlike
// __syncthreads() it does not wait for outstanding global loads (the staged direct-to-LDS loads of later steps).
__device__ __forceinline__ void lds_barrier() { __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// s_waitcnt vmcnt(n), other counters unconstrained (gfx9 encoding).
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

}  // namespace gfr
