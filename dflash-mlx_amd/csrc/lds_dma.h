// Direct global -> LDS loads with explicit waits, for kernels whose loader waves
// issue nothing else.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dflash {
namespace {

// The 32-bit LDS address of a workgroup-shared object.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// One direct global -> LDS load of 16 bytes a lane: lane l reads
// sbase + voff (its own byte offset) and its 16 bytes land at LDS address
// lds + 16 l.  Written as an instruction of its own so that the compiler
// does not see a pending LDS write and hold every later LDS read behind all
// of the loads in flight: the waits for these loads are explicit (wait_vm).
// M0 (the LDS base of the load) is set inside the instruction pair; the
// compiler treats M0 as reserved and does not use it in these kernels (the
// generated code's only M0 writes are these), so nothing it holds is lost.
__device__ __forceinline__ void dma16(const void* sbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(voff), "s"(sbase), "s"(lds) : "memory");
}

// The same with 4 bytes a lane, at lds + 4 l.
__device__ __forceinline__ void dma4(const void* sbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dword %0, %1"
               :: "v"(voff), "s"(sbase), "s"(lds) : "memory");
}

// Wait until at most N loads of this wave are outstanding (loads complete
// in issue order).
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The barrier of waves that read slots which loader waves refill behind it: their LDS
// reads are done.  (The products that use them are no memory operations, so the compiler
// may place these, and its own wait for the reads, on either side.)
__device__ __forceinline__ void read_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

}  // namespace
}  // namespace dflash
