// lds_dma.h -- global memory to LDS copies without registers, and the row swizzles
// of the GEMMs' stages (gfx950).
#ifndef SMAUL_LDS_DMA_H
#define SMAUL_LDS_DMA_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

// LDS rows keep their 16-byte chunks XOR-swizzled by row index, so the 32
// consecutive rows that one fragment read touches fall in distinct banks both
// for 32 banks read 8 lanes at a time and for 64 banks read 16 at a time.
__device__ __forceinline__ int swz_a(int r) { return (r & 6) | ((r ^ (r >> 3)) & 1); }        // 8 chunks
__device__ __forceinline__ int swz_b(int r) { return ((r >> 1) & 2) | (((r >> 1) ^ (r >> 3)) & 1); }  // 4

typedef __attribute__((address_space(3))) void* lds_vptr_t;

__device__ __forceinline__ uint32_t lds_offset(const void* p) { return (uint32_t)(uintptr_t)(lds_vptr_t)p; }

// LDS DMA: each lane copies 16 (or 4) bytes from base + off to LDS address
// lds + 16 (or 4) * lane.  Issued as inline asm so the compiler's wait-count
// pass does not treat every later LDS read as dependent on it (it cannot tell
// the stage buffers apart); the kernels wait for it explicitly (vmcnt) before
// the barrier that publishes a buffer.  M0 holds the LDS address (all 32 bits
// are used: addresses above 64 KB land where they should on gfx950); nothing
// else in these kernels uses M0.
// The base address is wave-uniform by construction; readfirstlane makes that
// explicit so it always lands in scalar registers.
__device__ __forceinline__ const void* uniform_ptr(const void* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const void*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(uniform_ptr(base)) : "memory");
}
__device__ __forceinline__ void dma4(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(uniform_ptr(base)) : "memory");
}
// wait until at most N of this wave's vector-memory loads are outstanding
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}

}  // namespace

#endif  // SMAUL_LDS_DMA_H
