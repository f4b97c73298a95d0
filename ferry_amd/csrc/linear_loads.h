// Loads of the linear products' kernels from memory straight to LDS, and their waits.
#pragma once

#include "linear.h"

#include <type_traits>

namespace ferry {
namespace lin {
namespace {

// A part of memory as a buffer: reads behind its end give 0, also into LDS.
__device__ __forceinline__ u32x4 buffer_at(const void* p, int64_t bytes) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const int64_t n = bytes < 0 ? 0 : (bytes > 0xffffffffll ? 0xffffffffll : bytes);
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) & 0xffffu,
               (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)n), 0x00020000u};
}
constexpr uint32_t kNowhere = 0xfffffff0u;   // an offset behind the end of every buffer

// (descriptors are wave-uniform, but the compiler may keep them in vector registers)
__device__ __forceinline__ u32x4 scalar(const u32x4& r) {
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)r[0]), (uint32_t)__builtin_amdgcn_readfirstlane((int)r[1]),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)r[2]), 0x00020000u};
}
// 16 bytes of each lane from offset soff + voff of the buffer to LDS address lds + 16 * lane; 0 from behind the
// buffer's end (soff itself must lie in it, or be 0: the hardware compares voff with size - soff).  Inline asm,
// so that no wait is added: their completion is awaited with wait_cnt.  m0 holds the LDS base; one wait state
// between its write and the load.
__device__ __forceinline__ void load_lds(u32x4 r, uint32_t voff, uint32_t soff, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %0, %1, %3 offen lds"
      :
      : "v"(voff), "s"(scalar(r)), "s"(__builtin_amdgcn_readfirstlane((int)lds)), "s"(__builtin_amdgcn_readfirstlane((int)soff))
      : "memory");
}
// 4 bytes of each lane, as above
__device__ __forceinline__ void load_lds4(u32x4 r, uint32_t voff, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %0, %1, 0 offen lds"
      :
      : "v"(voff), "s"(scalar(r)), "s"(__builtin_amdgcn_readfirstlane((int)lds))
      : "memory");
}
template <int VM>
__device__ __forceinline__ void wait_cnt() {   // at most VM loads and no LDS reads outstanding
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((VM & 15) | (7 << 4) | ((VM >> 4) << 14));
  asm volatile("" ::: "memory");
}
// no loads outstanding, in a form that the compiler counts with: loads to registers behind a condition would
// otherwise be waited for where the registers are written next, in the loop
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }
// no LDS reads outstanding
__device__ __forceinline__ void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (3 << 14));
  asm volatile("" ::: "memory");
}
// at most the loads of y chunks of L loads outstanding (values above V count as V)
template <int V, int L>
__device__ __forceinline__ void wait_chunks(int y) {
  if constexpr (V == 0) {
    wait_cnt<0>();
  } else {
    if (y >= V)
      wait_cnt<V * L>();
    else
      wait_chunks<V - 1, L>(y);
  }
}
// f(integral_constant<int, B>) ... f(integral_constant<int, E - 1>)
template <int B, int E, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (B < E) {
    f(std::integral_constant<int, B>{});
    static_for<B + 1, E>(f);
  }
}
// barrier of a workgroup without the fence of __syncthreads, which would drain the loads
__device__ __forceinline__ void wg_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

}  // namespace
}  // namespace lin
}  // namespace ferry
