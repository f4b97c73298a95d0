// What the expert FFN kernels share: the list of experts of a launch, direct global -> LDS loads and
// their waits, the table of row tiles of a list.
#pragma once

#include "common.h"

namespace ferry {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kListMax = 256;   // experts per launch (longer lists are split by the host)

struct ExpertList {
  int32_t n;
  int32_t n_mid;   // small-expert up launch: the first n_mid entries take 64-column workgroups
  int16_t expert[kListMax];
  int32_t slot[kListMax];
};

__device__ __forceinline__ float silu_mul(float g, float u) {
  // silu(g) * u in fp32 on the up projections' results: g * u / (1 + e^-g) with the
  // hardware exp2 and reciprocal (relative error ~1e-6, far below the bf16 rounding that
  // follows); a large negative g gives e^-g = inf and a zero result, the exact formula's limit
  return g * u * __builtin_amdgcn_rcpf(1.0f + __expf(-g));
}

// two floats rounded to bf16 (round to nearest even, as f32_to_bf16) in one instruction,
// packed as lo | hi << 16
__device__ __forceinline__ uint32_t pk_bf16(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, b16x2));
}

// =============================================================================================
// Memory helpers shared by the kernels below
// =============================================================================================

// a wave-uniform value / pointer moved to scalar registers
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
template <typename T>
__device__ __forceinline__ const T* uniform_ptr(const T* p) {
  return (const T*)(uintptr_t)uniform64((int64_t)(uintptr_t)p);
}
// 16-byte global->LDS direct load of each lane: global address sbase + voff (wave-uniform base
// in scalar registers, 32-bit lane byte offset), LDS byte address lds + 16 * lane.  Issued as
// inline asm so that the address keeps this form wherever the load is scheduled; the compiler
// does not track these loads, their completion is awaited with wait_cnt / wait_vmcnt.  The asm writes
// m0 (the LDS base of the direct load); nothing else in these kernels uses m0.  An LDS direct
// load needs one wait state between the SALU write of m0 and its issue (the s_nop), which the
// compiler's hazard pass would add for its own instructions but cannot see inside the asm.
__device__ __forceinline__ void dma16(const char* sbase, uint32_t voff, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(voff), "s"(sbase), "s"(lds)
      : "memory", "m0");
}

typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(lds_char*)p;
}
// 4-byte global->LDS direct load of each lane (LDS byte address lds + 4 * lane), as dma16
__device__ __forceinline__ void dma4(const char* sbase, uint32_t voff, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %0, %1"
      :
      : "v"(voff), "s"(sbase), "s"(lds)
      : "memory", "m0");
}
// 2-byte load of each lane, zero-extended to 4 bytes in LDS (address lds + 4 * lane)
__device__ __forceinline__ void dma2(const char* sbase, uint32_t voff, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_ushort %0, %1"
      :
      : "v"(voff), "s"(sbase), "s"(lds)
      : "memory", "m0");
}
// 16 bytes at LDS byte address addr (constant parts of it go into the instruction's offset)
__device__ __forceinline__ bf16x8 lds_read16(uint32_t addr) {
  return *reinterpret_cast<__attribute__((address_space(3))) const bf16x8*>((uintptr_t)addr);
}
// wait until at most VM vector-memory operations (the direct loads among them) and no LDS reads
// of this wavefront are outstanding, in a form whose LDS part the compiler knows of
template <int VM>
__device__ __forceinline__ void wait_cnt() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((VM & 15) | (7 << 4) | ((VM >> 4) << 14));
  asm volatile("" ::: "memory");
}
// workgroup barrier without the release/acquire fence of __syncthreads (which would drain
// the direct loads of the later stages); LDS visibility is established by the explicit waits
__device__ __forceinline__ void wg_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

struct TileTable {
  __attribute__((aligned(16))) int32_t cum[kListMax + 1];  // cumulative M tiles over list entries
  int32_t total;
  int64_t start[kListMax];    // per list entry: its expert's first grouped row, and row count
  int32_t rows[kListMax];
};

// Wavefront 0 builds the cumulative counts of M tiles of `rows` rows of the listed experts with more than
// LEAST rows.
template <int LEAST, typename Args>
__device__ __forceinline__ void build_tile_table(const Args& a, TileTable& tt, uint32_t rows) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int cnt[4];
    int local = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int li = lane * 4 + q;
      int c = 0;
      if (li < a.list.n) {
        const int e = a.list.expert[li];
        const int64_t s0 = a.starts[e];
        const int64_t n = a.starts[e + 1] - s0;
        c = n > LEAST ? (int)(((uint32_t)n + rows - 1) / rows) : 0;
        tt.start[li] = s0;
        tt.rows[li] = (int32_t)n;
      }
      cnt[q] = c;
      local += c;
    }
    int incl = local;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(incl, off, 64);
      if (lane >= off) incl += v;
    }
    int run = incl - local;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      tt.cum[lane * 4 + q] = run;
      run += cnt[q];
    }
    if (lane == 63) {
      tt.cum[kListMax] = incl;
      tt.total = incl;
    }
  }
  __syncthreads();
}

// largest li with cum[li] <= m (cum is non-decreasing), by a whole wavefront: the entries that hold
// at most m, counted with ballots over four entries a lane
__device__ __forceinline__ int find_entry(const TileTable& tt, int m) {
  const u32x4 c = *reinterpret_cast<const u32x4*>(&tt.cum[(threadIdx.x & 63) * 4]);
  int le = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) le += __popcll(__ballot((int)c[q] <= m));
  return le - 1;
}

}  // namespace
}  // namespace ferry
