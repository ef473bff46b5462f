// Asynchronous loads straight into LDS whose waits are the kernel's own. (The builtin's are counted by the compiler,
// which then waits for every one of them before any LDS read that follows, whichever tile it is of.)
#pragma once

#include "dsa_common.h"

namespace dsa {

// The LDS address of a shared object, for the loads below (wave-uniform).
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane(
      (int)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}

// 16 bytes from each lane's address into LDS at lds + 16 x lane. Nothing waits for it: s_waitcnt vmcnt before the barrier
// that hands the data on (the loads of a wave end in order, and count with its other global accesses). m0, the LDS
// address, is an operand, so that the compiler knows of its value; a scalar write of it needs one wait state before the
// load, which the compiler does not see in here and may leave no other instruction for.
__device__ __forceinline__ void load_lds16(const void* p, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "{m0}"(lds) : "memory");
}

// At most N of the wave's global accesses are still out (loads end in order).
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A barrier of the whole workgroup: its LDS accesses before it are visible after it, global loads stay in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The lane, as a value that the compiler knows nothing about: what is computed from it stays where it is used instead
// of being carried in registers around a loop.
__device__ __forceinline__ int fresh_lane() {
  int x = threadIdx.x & (WAVE - 1);
  asm volatile("" : "+v"(x));
  return x;
}

// Loads into registers are complete after this (waited for here, not at a use inside a loop).
template <typename T, int N>
__device__ __forceinline__ void arrive(T (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

}  // namespace dsa
