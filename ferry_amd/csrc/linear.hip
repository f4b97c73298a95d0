// Dense and expert-grouped linear products with their epilogue and gradients: the kernels that take
// every size and alignment, and the entry points.  No counterpart in the reference, whose experts are
// SwiGLU blocks of bf16 matrices without biases or gradients.
#include "linear.h"
#include "linear_plan.h"
#include "linear_tile.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace ferry {
namespace lin {
namespace {

// =============================================================================================
// Any size, any alignment
// =============================================================================================

// eight 16-bit values from p, of which the first n are there (the others 0).  p may lie at any even
// address: the hardware takes unaligned 16-byte loads.
__device__ __forceinline__ u32x4 load8(const uint16_t* p, int n) {
  u32x4 v = {0, 0, 0, 0};
  if (n >= 8) {
    __builtin_memcpy(&v, p, 16);
  } else if (n > 0) {
    uint16_t h[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) h[q] = q < n ? p[q] : (uint16_t)0;
    __builtin_memcpy(&v, h, 16);
  }
  return v;
}

// TI x TJ outputs per workgroup of four wavefronts, 64 of the contraction a step through registers into one of two
// LDS buffers, the loads of a step issued before the products of the one before.  (Loads two steps ahead took 300
// registers, one wavefront a SIMD: dx of 8,192 x 6,143 x 2,047 in 1,007 us instead of 614.)  Loads are
// 16 bytes at any alignment; what lies outside the matrices, the group or the contraction is 0 in LDS, so
// that nothing a neighbouring row holds, a NaN included, enters a sum.
template <typename T, int MODE, int TI, int TJ>
__global__ __launch_bounds__(256) void any_kernel(Args a) {
  constexpr bool kAcrossA = MODE == kDw, kAcrossB = MODE != kFwd, kRaggedI = MODE != kDw;
  constexpr int kStage = (TI + TJ) * 128, MI = TI / 32, NJ = TJ / 32;
  __shared__ Table tt;
  __shared__ int32_t first_s[kMaxGroups];
  __shared__ __attribute__((aligned(1024))) char smem[2 * kStage];
  const int ntj = (int)ceil_div(a.J, TJ);
  const int nti = kRaggedI ? 0 : (int)ceil_div(a.I, TI);
  build_table<kRaggedI>(a, tt, kRaggedI ? TI : nti, first_s);
  if (a.zero_rest) zero_rest(a, tt.first, tt.last);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = (wave >> 1) * (TI / 2), wj = (wave & 1) * (TJ / 2);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  const int64_t total = (int64_t)tt.total * ntj * a.splits;
  for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
    const int s = (int)(item % a.splits);
    const int64_t t = item / a.splits;
    const int jt = (int)(t % ntj), mt = (int)(t / ntj);
    const int g = a.starts ? find_group(tt, mt) : 0;
    const int64_t start = first_s[g], n = tt.rows[g];
    const int64_t i0 = (int64_t)(mt - tt.cum[g]) * TI, j0 = (int64_t)jt * TJ;
    const int64_t I = kRaggedI ? n : a.I, C = kRaggedI ? a.C : n;
    const int64_t per = ceil_div(ceil_div(C, a.splits), 64) * 64;
    const int64_t c0 = s * per, c1 = c0 + per < C ? c0 + per : C;
    const uint16_t* const bw = a.b + (MODE == kDw ? 0 : g * a.b_group);
    // operands by index: each thread's rows
    const uint16_t* pa[MI];
    const uint16_t* pb[NJ];
    if constexpr (!kAcrossA) {
#pragma unroll
      for (int q = 0; q < MI; ++q) {
        const int64_t i = i0 + tid / 8 + 32 * q;
        int64_t r = start + i;
        bool ok = i < I;
        if (MODE == kFwd && a.rows && ok) {
          r = a.rows[r];
          ok = (uint64_t)r < (uint64_t)a.x_rows;
        }
        pa[q] = ok ? a.a + r * a.lda + (tid & 7) * 8 : nullptr;
      }
    }
    if constexpr (!kAcrossB) {
#pragma unroll
      for (int q = 0; q < NJ; ++q) {
        const int64_t j = j0 + tid / 8 + 32 * q;
        pb[q] = j < a.J ? bw + j * a.ldb + (tid & 7) * 8 : nullptr;
      }
    }
    u32x4 va[MI], vb[NJ];
    auto load = [&](int64_t c) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < MI; ++q) {
        if constexpr (!kAcrossA) {
          va[q] = load8(pa[q] + c, pa[q] ? (int)(c1 - c < 64 ? c1 - c : 64) - (tid & 7) * 8 : 0);
        } else {
          constexpr int per_row = TI / 8;
          const int64_t cc = c + tid / per_row + (256 / per_row) * q, i = i0 + (tid % per_row) * 8;
          va[q] = load8(a.a + (start + cc) * a.lda + i, cc < c1 ? (int)(I - i < 8 ? I - i : 8) : 0);
        }
      }
#pragma unroll
      for (int q = 0; q < NJ; ++q) {
        if constexpr (!kAcrossB) {
          vb[q] = load8(pb[q] + c, pb[q] ? (int)(c1 - c < 64 ? c1 - c : 64) - (tid & 7) * 8 : 0);
        } else {
          constexpr int per_row = TJ / 8;
          const int64_t cc = c + tid / per_row + (256 / per_row) * q, j = j0 + (tid % per_row) * 8;
          int64_t r = cc;
          bool ok = cc < c1;
          if (MODE == kDw && ok) {
            r = start + cc;
            if (a.rows) {
              r = a.rows[r];
              ok = (uint64_t)r < (uint64_t)a.x_rows;
            }
          }
          vb[q] = load8(bw + (ok ? r * a.ldb : 0) + j, ok ? (int)(a.J - j < 8 ? a.J - j : 8) : 0);
        }
      }
    };
    auto store = [&](int buf) __attribute__((always_inline)) {
      char* const st = smem + buf * kStage;
#pragma unroll
      for (int q = 0; q < MI; ++q) {
        constexpr int per_row = kAcrossA ? TI / 8 : 8;
        const int r = tid / per_row + (256 / per_row) * q, k = tid % per_row;
        const int at = kAcrossA ? r * TI * 2 + ((k ^ swz_across<TI>(r)) << 4) : r * 128 + ((k ^ swz_direct(r)) << 4);
        *reinterpret_cast<u32x4*>(st + at) = va[q];
      }
#pragma unroll
      for (int q = 0; q < NJ; ++q) {
        constexpr int per_row = kAcrossB ? TJ / 8 : 8;
        const int r = tid / per_row + (256 / per_row) * q, k = tid % per_row;
        const int at = kAcrossB ? r * TJ * 2 + ((k ^ swz_across<TJ>(r)) << 4) : r * 128 + ((k ^ swz_direct(r)) << 4);
        *reinterpret_cast<u32x4*>(st + TI * 128 + at) = vb[q];
      }
    };
    f32x4 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    __syncthreads();   // the tile before has read its last buffer
    auto products = [&](int buf) __attribute__((always_inline)) {
      const uint32_t la = lds0 + buf * kStage, lb = la + TI * 128;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        s16x8 fa[MI], fb[NJ];
#pragma unroll
        for (int i = 0; i < MI; ++i)
          fa[i] = kAcrossA ? read_across(la + frag_across<TI>(wi + 16 * i, ks, 0), la + frag_across<TI>(wi + 16 * i, ks, 1))
                           : read_direct(la + frag_direct(wi + 16 * i, ks));
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          fb[j] = kAcrossB ? read_across(lb + frag_across<TJ>(wj + 16 * j, ks, 0), lb + frag_across<TJ>(wj + 16 * j, ks, 1))
                           : read_direct(lb + frag_direct(wj + 16 * j, ks));
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = T::mma(fb[j], fa[i], acc[i][j]);
      }
    };
    load(c0);
    store(0);
    int buf = 0;
    for (int64_t c = c0; c < c1; c += 64, buf ^= 1) {
      const bool more = c + 64 < c1;
      if (more) load(c + 64);
      __syncthreads();
      products(buf);
      if (more) store(buf ^ 1);
    }
    // lane l holds columns 4 (l / 16) + [0, 4) of row l % 16 of each 16 x 16 tile
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int64_t r = i0 + wi + 16 * i + (lane & 15);
      if (r >= I) continue;
      const int64_t row = kRaggedI ? start + r : r;
#pragma unroll
      for (int jj = 0; jj < NJ; ++jj) {
        const int64_t j = j0 + wj + 16 * jj + 4 * (lane >> 4);
        const int m = (int)(a.J - j < 4 ? a.J - j : 4);
        if (m <= 0) continue;
        if (a.splits > 1) {
          float* const o = a.part + (kRaggedI ? (s * a.pairs + row) : ((int64_t)s * a.groups + g) * a.I + row) * a.J + j;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q < m) o[q] = acc[i][jj][q];
        } else if constexpr (MODE == kDw) {
          Args d = a;
          d.out = a.out + g * a.o_group;
          finish4<T>(d, g, row, j, m, acc[i][jj]);
        } else {
          finish4<T>(a, g, row, j, m, acc[i][jj]);
        }
      }
    }
  }
}

// The parts of a split contraction added in their order, and the epilogue.  A wavefront takes 256
// columns of a row.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t per = ceil_div(a.J, 256), rows = MODE == kDw ? a.groups * a.I : a.pairs, items = rows * per;
  for (int64_t it = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += (int64_t)gridDim.x * 4) {
    const int64_t row = it / per, j = (it % per) * 256 + lane * 4;
    if (j >= a.J) continue;
    const int m = (int)(a.J - j < 4 ? a.J - j : 4);
    int g = MODE == kDw ? (int)(row / a.I) : 0;
    bool in = true;
    if (MODE != kDw && a.starts) {
      in = false;
      for (int k = 0; k < a.groups && !in; ++k)
        if (row >= group_start(a, k) && row < group_start(a, k + 1)) g = k, in = true;
    }
    Args d = a;
    if (MODE == kDw) d.out = a.out + g * a.o_group;
    const int64_t orow = MODE == kDw ? row % a.I : row;
    if (!in) {
      if (a.zero_rest)
        for (int q = 0; q < m; ++q) a.out[row * a.ldo + j + q] = 0;
      continue;
    }
    f32x4 v = {0, 0, 0, 0};
    for (int s = 0; s < a.splits; ++s) {
      const float* const p = a.part + (s * rows + row) * a.J + j;
      if (m == 4 && a.J % 4 == 0) {
        v += *reinterpret_cast<const f32x4*>(p);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += q < m ? p[q] : 0.f;
      }
    }
    finish4<T>(d, g, orow, j, m, v);
  }
}

// =============================================================================================
// The epilogue's gradient, and sums
// =============================================================================================

struct SlopeArgs {
  const uint16_t* dy;
  const uint16_t* pre;   // act != 0
  uint16_t* dz;          // null: not wanted (act == 0)
  uint16_t* db;          // null: not wanted; [groups][N]
  float* part;           // [splits][groups][N], with splits > 1
  int64_t ldy, pairs, N;
  const int64_t* starts;
  int32_t groups, splits, act;
};

// f[q] = f'(f[q]), the choice of the activation once for eight
__device__ __forceinline__ void slope8(int act, float (&f)[8]) {
  auto all = [&](auto a) {
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = slope(decltype(a)::value, f[q]);
  };
  switch (act) {
    case kRelu: return all(std::integral_constant<int, kRelu>{});
    case kSilu: return all(std::integral_constant<int, kSilu>{});
    case kGelu: return all(std::integral_constant<int, kGelu>{});
    default: return all(std::integral_constant<int, kGeluTanh>{});
  }
}

// dz = dy f'(pre) rounded, and db = the sum of the unrounded dz over each group's rows.  A workgroup takes
// 2048 / RL columns (8 a thread) of one part of a group's rows, RL rows side by side and four of those at a
// time, whose loads are issued together.  Large calls are bound by memory (dy and pre in, dz out) and take RL = 8
// and parts, which a second launch adds; small ones by the chain of loads of a column's rows, which RL = 32 and, where
// columns are few, 128 shorten without parts (300 rows of 2,816: 15 + 4 us with parts, 7 with RL = 128).
template <typename T, int RL>
__global__ __launch_bounds__(256) void slope_kernel(SlopeArgs a) {
  constexpr int CL = 256 / RL, COLS = CL * 8, U = 4;
  __shared__ float sum[4][COLS];
  const int tid = threadIdx.x, rl = tid / CL, cl = (tid % CL) * 8;
  const int64_t jb = ceil_div(a.N, COLS), items = jb * a.groups * a.splits;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t j = (it % jb) * COLS + cl;
    const int g = (int)(it / jb % a.groups), s = (int)(it / jb / a.groups);
    int64_t lo = 0, hi = a.pairs;
    if (a.starts) {
      lo = a.starts[g];
      hi = a.starts[g + 1];
      lo = lo < 0 ? 0 : (lo > a.pairs ? a.pairs : lo);
      hi = hi < lo ? lo : (hi > a.pairs ? a.pairs : hi);
    }
    const int64_t per = ceil_div(hi - lo, a.splits);
    const int64_t r0 = lo + s * per, r1 = r0 + per < hi ? r0 + per : hi;
    const int m = (int)(a.N - j < 8 ? a.N - j : 8);
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (m > 0)
      for (int64_t rr = r0 + rl; rr < r1; rr += U * RL) {
        u32x4 y[U], z[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t r = rr + u * RL;
          y[u] = load8(a.dy + r * a.ldy + j, r < r1 ? m : 0);
          z[u] = load8(a.pre + r * a.N + j, a.act != kNone && r < r1 ? m : 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t r = rr + u * RL;
          if (r >= r1) continue;
          float v[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = T::load((uint16_t)(y[u][q >> 1] >> (16 * (q & 1))));
          if (a.act != kNone) {
            float f[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) f[q] = T::load((uint16_t)(z[u][q >> 1] >> (16 * (q & 1))));
            slope8(a.act, f);
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] *= f[q];
            uint16_t* const o = a.dz + r * a.N + j;
            u32x4 w;
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = T::round2(v[2 * q], v[2 * q + 1]);
            if (m == 8) {
              __builtin_memcpy(o, &w, 16);
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                if (q < m) o[q] = (uint16_t)(w[q >> 1] >> (16 * (q & 1)));
            }
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) acc[q] += v[q];
        }
      }
    if (!a.db) continue;
    // the lanes of a wavefront that hold the same columns, then the wavefronts
#pragma unroll
    for (int off = CL; off < 64; off <<= 1)
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += __shfl_xor(acc[q], off, 64);
    __syncthreads();
    if ((tid & 63) < CL) {
#pragma unroll
      for (int q = 0; q < 8; ++q) sum[tid >> 6][cl + q] = acc[q];
    }
    __syncthreads();
    const int64_t jj = (it % jb) * COLS + tid;
    if (tid < COLS && jj < a.N) {
      const float t = (sum[0][tid] + sum[1][tid]) + (sum[2][tid] + sum[3][tid]);
      if (a.splits > 1)
        a.part[((int64_t)s * a.groups + g) * a.N + jj] = t;
      else
        a.db[(int64_t)g * a.N + jj] = T::round(t);
    }
  }
}

// The parts' sums: 64 columns a workgroup, each wavefront every fourth part, eight loads at a time.
template <typename T>
__global__ __launch_bounds__(256) void slope_join_kernel(const float* __restrict__ part, int64_t n, int splits,
                                                         uint16_t* __restrict__ db) {
  __shared__ float sum[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t i0 = (int64_t)blockIdx.x * 64; i0 < n; i0 += (int64_t)gridDim.x * 64) {
    const int64_t i = i0 + lane < n ? i0 + lane : n - 1;
    float t = 0;
#pragma unroll 8
    for (int s = wave; s < splits; s += 4) t += part[s * n + i];
    sum[wave][lane] = t;
    __syncthreads();
    if (wave == 0 && i0 + lane < n) db[i] = T::round((sum[0][lane] + sum[1][lane]) + (sum[2][lane] + sum[3][lane]));
    __syncthreads();
  }
}

// out[t] = sum over j ascending of part[pair_pos[t, j]], fp32, rounded once; entries outside the pairs
// add nothing.  Bound by reading part.
template <typename T>
__global__ __launch_bounds__(256) void sum_pairs_kernel(const uint16_t* __restrict__ part, int64_t pairs, int64_t K,
                                                        int64_t ldp, const int32_t* __restrict__ pos, int64_t tokens,
                                                        int topk, uint16_t* __restrict__ out) {
  const int64_t per = ceil_div(K, 8), items = tokens * per;
  for (int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x; it < items; it += (int64_t)gridDim.x * 256) {
    const int64_t t = it / per, k = (it % per) * 8;
    const int m = (int)(K - k < 8 ? K - k : 8);
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
    for (int j = 0; j < topk; ++j) {
      const int32_t p = pos[t * topk + j];
      if ((uint32_t)p < (uint64_t)pairs) {
        const u32x4 v = load8(part + p * ldp + k, m);
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] += T::load((uint16_t)(v[q >> 1] >> (16 * (q & 1))));
      }
    }
    u32x4 w;
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = T::round2(acc[2 * q], acc[2 * q + 1]);
    uint16_t* const o = out + t * K + k;
    if (m == 8) {
      __builtin_memcpy(o, &w, 16);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < m) o[q] = (uint16_t)(w[q >> 1] >> (16 * (q & 1)));
    }
  }
}

// =============================================================================================
// Host
// =============================================================================================

int64_t cus() {   // of the current device
  static int64_t known[64];
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!known[dev]) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return 256;
    known[dev] = n;
  }
  return known[dev];
}

// Parts of the contraction for any_kernel: as many as give every CU a tile, of at least 256 each.
int64_t splits_of(int64_t tiles, int64_t c) {
  const int64_t want = tiles > 0 ? 256 / tiles : 1, most = c / 256;
  return std::max<int64_t>(1, std::min<int64_t>({want, most, 32}));
}

enum Kind { kAny = 0, kTiles = 1, kFew = 2 };
struct Plan {
  Kind kind;
  int shape;      // kTiles: 0 256 x 256, 1 .. 4 of ring_launch
  int mt, nb;     // kFew: rows and columns of a tile in 16s
  int any;        // rows and columns of any_kernel's tile
  int64_t tiles;  // upper bound (kFew: of row tiles, with one of splits)
  int64_t splits;
};

// The tiles' sizes (indices of A and of B), and their time in us: for a stage of 64 of the contraction, and for
// what a tile costs besides.  Measured at 8,192 x 6,144 x 2,048 and its gradients.
struct TileCost {
  int tm, tn;
  double stage, fixed;
};
const TileCost kShapes[] = {{256, 256, 1.31, 6.0}, {256, 128, 1.04, 4.0}, {128, 128, 0.58, 3.0}, {64, 128, 0.40, 2.5}, {64, 64, 0.32, 2.0}};
// few_kernel's tiles in 16s, wavefronts, workgroups resident on a CU, us for a step of 64 of the contraction a wavefront
struct FewCost {
  int mt, nb, waves, resident;
  double step;
};
const FewCost kFews[] = {{1, 1, 8, 1, 0.36}, {1, 1, 4, 2, 0.34}, {1, 2, 4, 2, 0.46}, {2, 2, 4, 2, 0.42}, {4, 2, 4, 1, 0.65}, {4, 4, 4, 1, 0.85}};
constexpr double kLaunch = 3.5;    // us until the first products of a launch, and for its end
constexpr double kMemory = 4.8e6;  // bytes a us

// op: the product; rows: pairs
Plan make_plan(int op, int64_t pairs, int64_t n, int64_t k, int64_t groups, int64_t cu) {
  Plan p = {};
  const int64_t J = op == kFwd ? n : k, used = std::min(groups, std::max<int64_t>(pairs, 1));
  auto row_tiles = [&](int64_t t) { return ceil_div(pairs, t) + (groups > 1 ? used : 0); };
  auto tiles = [&](int64_t tm, int64_t tn) { return (op == kDw ? groups * ceil_div(n, tm) : row_tiles(tm)) * ceil_div(J, tn); };
  p.any = tiles(128, 128) >= 512 ? 128 : 64;
  p.splits = 1;
  const double c = op == kFwd ? (double)k : (op == kDx ? (double)n : (double)pairs / (double)groups);
  const bool tiled = n % 8 == 0 && k % 8 == 0, few = op == kDx ? tiled && groups == 1 : op == kFwd && k % 8 == 0 && (groups == 1 || pairs <= 6 * used);
  if (!tiled && !few) {
    p.tiles = tiles(p.any, p.any);
    p.splits = splits_of(p.tiles, (int64_t)c);
    return p;
  }
  // The cheapest kernel, tile and number of parts: whole rounds of tiles over the CUs (of groups of unknown sizes, as
  // many tiles as equal ones and half a tile of each group), no faster than the operands come from memory, the
  // parts' way through memory, and for groups half a tile's time until the last is done.
  const double rows = (double)pairs / used, out = (double)(op == kDw ? groups * n * k : pairs * J);
  const double bytes = 2.0 * (op == kDw ? (double)pairs * (n + k) + out : (double)pairs * (n + k) + (double)used * n * k);
  auto m_tiles = [&](int tm) {
    if (op == kDw) return (double)(groups * ceil_div(n, tm));
    return groups > 1 ? used * std::max(1.0, rows / tm + 0.5) : (double)ceil_div(pairs, tm);
  };
  auto time = [&](double items, double slots, double item) {
    const double rounds = groups > 1 ? std::max(1.0, items / slots) : std::ceil(items / slots);
    return kLaunch + std::max(rounds * item, bytes / kMemory) + (groups > 1 ? 0.5 * item : 0.0);
  };
  double least = 1e30;
  if (few)
    for (const FewCost& f : kFews) {
      // kDx loads w by pieces of its rows, and of groups tiles of 32 x 32 were the fastest
      if ((op == kDx && f.mt != f.nb) || (op == kDx && f.mt == 1) || (groups > 1 && f.mt != 2)) continue;
      const double items = m_tiles(16 * f.mt) * ceil_div(J, 16 * f.nb);
      if (f.nb == 1 && (f.waves == 8) != (row_tiles(16) * ceil_div(J, 16) <= cu)) continue;   // as few_launch has it
      const double step = f.step * (op == kDx && f.nb == 2 ? 1.5 : 1.0);
      const double cost = time(items, (double)cu * f.resident, (1.0 + std::ceil(c / (64 * f.waves)) * step) * (groups > 1 ? 1.5 : 1.0));
      if (cost < least) {
        least = cost;
        p.kind = kFew;
        p.mt = f.mt;
        p.nb = f.nb;
      }
    }
  if (tiled)
    for (int i = 0; i < 5; ++i) {
      const TileCost& t = kShapes[i];
      for (int64_t parts = 1; parts <= 16; parts *= 2) {
        if (parts > 1 && c / parts < 256) break;
        // (groups' small tiles share less of the operands in L2)
        const double stage = t.stage * (groups > 1 && t.tm == 64 ? 1.4 : 1.0);
        double cost = time(m_tiles(t.tm) * ceil_div(J, t.tn) * parts, (double)cu, std::ceil(c / 64 / parts) * stage + t.fixed);
        if (parts > 1) cost += 4.0 + out * (8.0 * parts + 2.0) / kMemory;
        if (cost < least) {
          least = cost;
          p.kind = kTiles;
          p.shape = i;
          p.splits = parts;
        }
      }
    }
  p.tiles = p.kind == kFew ? row_tiles(16 * p.mt) : tiles(kShapes[p.shape].tm, kShapes[p.shape].tn);
  return p;
}

// make_plan for the current device; a thread keeps its latest plans, by the sizes they depend on
Plan plan(int op, int64_t pairs, int64_t n, int64_t k, int64_t groups) {
  struct Kept {
    int64_t key[6];
    Plan plan;
  };
  static thread_local Kept kept[16];
  const int64_t key[6] = {op + 1, pairs, n, k, groups, cus()};
  uint64_t h = 0;
  for (int64_t v : key) h = (h ^ (uint64_t)v) * 0x9e3779b97f4a7c15ull;
  Kept& e = kept[h >> 60];
  if (!std::equal(key, key + 6, e.key)) {
    e.plan = make_plan(op, pairs, n, k, groups, key[5]);
    std::copy(key, key + 6, e.key);
  }
  return e.plan;
}

bool even(const void* q, int64_t stride) { return (uintptr_t)q % 16 == 0 && stride % 8 == 0; }

// Whether few_kernel can read the operands: rows at multiples of 16 bytes, offsets that 32 bits hold.
bool few_fits(int op, const Args& a) {
  const int64_t most = ((int64_t)1 << 31) - (1 << 20);
  return a.C % 8 == 0 && (op == kFwd || a.J % 8 == 0) && even(a.a, a.lda) && even(a.b, a.ldb) && a.b_group % 8 == 0 &&
         a.ldb <= most / 128 && a.lda <= most / 128 && a.C <= most / 4 && (op == kFwd || (a.C + 128) * a.ldb <= most) &&
         (!a.rows || (a.x_rows >= 1 && a.x_rows * a.lda <= most));
}

// Whether the tiled kernels can read and write the operands: rows at multiples of 16 bytes, offsets that 32
// bits hold (a tile's, or all of an operand whose rows are gathered or follow the contraction).  Their forms for
// gathered rows add a bias and no more: expert_linear asks for nothing else, and any_kernel takes the C entry's other calls.
bool tiles_fit(int op, const Args& a, int64_t pairs, int64_t n, int64_t k) {
  if (a.rows && (a.x_rows < 1 || a.act != kNone || a.residual || a.pre)) return false;
  if (n % 8 || k % 8 || !even(a.a, a.lda) || !even(a.b, a.ldb) || a.b_group % 8 || !even(a.out, a.ldo) || a.o_group % 8 ||
      (a.bias && !even(a.bias, a.bias_group)) || (a.residual && !even(a.residual, a.ldr)) || (a.pre && !even(a.pre, 0)))
    return false;
  const int64_t most = ((int64_t)1 << 31) - (1 << 20);   // elements, with room for a stage behind the end
  const int64_t ia = op == kDw ? pairs : (a.rows ? a.x_rows : 512), ib = op == kFwd ? 512 : (op == kDx ? n : (a.rows ? a.x_rows : pairs));
  return a.J <= most / 1024 && a.lda <= most / 512 && a.ldb <= most / 512 && a.ldo <= most / 512 && a.ldr <= most / 512 && ia * a.lda <= most &&
         ib * a.ldb <= most && a.C <= most / 4;
}

int64_t part_bytes(int op, const Plan& p, int64_t pairs, int64_t n, int64_t k, int64_t groups) {
  if (p.splits <= 1) return 0;
  const int64_t out = op == kDw ? groups * n * k : pairs * (op == kFwd ? n : k);
  return p.splits * out * 4;
}

// Parts of a group's rows for slope_kernel, 1: all rows by one workgroup, 32 or 128 side by side.  Few rows take one
// launch without parts (300 rows of 2,816: 15 + 4 us with parts of 60 rows, 7 without).  Otherwise a part for each 128
// rows of a group on average, and for each 8,192 of the call, since one group may hold most of them; 64 at most (65,536
// rows of 1,536 in 128 equal groups: 38 us, 33 without; all of them in one group: 254, 449 without).
int64_t slope_splits(int64_t pairs, int64_t groups) {
  const int64_t rows = pairs / groups;
  return rows <= 512 && pairs <= 8192 ? 1 : std::min<int64_t>(std::max(ceil_div(rows, 128), ceil_div(pairs, 8192)), 64);
}

template <typename T, int MODE>
int run_typed(const Args& a, const Plan& p, int64_t n, int64_t k, hipStream_t s) {
  static const char* const names[] = {"linear_fwd", "linear_dx", "linear_dw"};
  // (tile256 keeps pre beside an activation only)
  const bool ring = MODE == kFwd && (a.rows ? !tile256_gathers(k, a.splits) : a.pre && a.act == kNone);
  const int shape = p.shape == 0 && ring ? 1 : p.shape;
  if (p.kind == kFew && few_fits(MODE, a)) {
    few_launch(MODE, T::kType, p.mt, p.nb, a, p.tiles, cus(), s);
  } else if (p.kind == kTiles && tiles_fit(MODE, a, a.pairs, n, k)) {
    if (shape == 0)
      tile_launch(MODE, T::kType, names[MODE], a, p.tiles * p.splits, cus(), s);
    else
      ring_launch(MODE, T::kType, shape, names[MODE], a, std::max(p.tiles * p.splits, shape == p.shape ? 0 : cus()), cus(), s);
  } else {
    const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>(p.tiles * p.splits * (p.kind == kFew ? 8 : 4), cus() * 4)));
    if (p.any == 128)
      launch(names[MODE], any_kernel<T, MODE, 128, 128>, grid, dim3(256), 0, s, a);
    else
      launch(names[MODE], any_kernel<T, MODE, 64, 64>, grid, dim3(256), 0, s, a);
  }
  FERRY_LAUNCHED(names[MODE]);
  if (a.splits > 1) {
    const int64_t rows = MODE == kDw ? a.groups * a.I : a.pairs;
    launch("linear_join", join_kernel<T, MODE>,
           dim3((unsigned)std::min<int64_t>(ceil_div(rows * ceil_div(a.J, 256), 4), 65536)), dim3(256), 0, s, a);
    FERRY_LAUNCHED("linear_join");
  }
  return 0;
}

template <int MODE>
int run(Args& a, int32_t dtype, int64_t pairs, int64_t n, int64_t k, void* workspace, int64_t workspace_bytes,
        hipStream_t s) {
  const Plan p = plan(MODE, pairs, n, k, a.groups);
  const int64_t need = part_bytes(MODE, p, pairs, n, k, a.groups);
  FERRY_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), "workspace too small (%lld < %lld bytes)",
                  (long long)workspace_bytes, (long long)need);
  FERRY_CHECK_ARG(need == 0 || (uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
  a.pairs = pairs;
  a.splits = (int32_t)p.splits;
  a.part = (float*)workspace;
  auto even = [](const void* q, int64_t stride) { return (uintptr_t)q % 8 == 0 && stride % 4 == 0; };
  a.vec_out = even(a.out, a.ldo) && a.o_group % 4 == 0 && (!a.residual || even(a.residual, a.ldr)) &&
              (!a.pre || even(a.pre, a.J));
  return dtype == FERRY_BF16 ? run_typed<Bf16, MODE>(a, p, n, k, s) : run_typed<F16, MODE>(a, p, n, k, s);
}

// The distance of rows whose stride a call with one of them need not name: the tiled kernels tell rows that are not there by
// offsets behind the end of the last one.
int64_t row_stride(int64_t stride, int64_t rows, int64_t width) { return rows > 1 ? stride : std::max(stride, width); }

constexpr int64_t kMost = (int64_t)1 << 30;   // rows, columns, pairs: tile numbers are counted in 32 bits

int check_sizes(int32_t dtype, int64_t pairs, int64_t n, int64_t k, int64_t groups, const int64_t* starts) {
  FERRY_CHECK_ARG(dtype == FERRY_BF16 || dtype == FERRY_F16, "dtype must be bf16 or fp16");
  FERRY_CHECK_ARG(pairs >= 0 && pairs < kMost && n >= 1 && n < kMost && k >= 1 && k < kMost,
                  "bad sizes: rows in [0, 2^30), n and k in [1, 2^30)");
  FERRY_CHECK_ARG(groups >= 1 && groups <= kMaxGroups, "groups must be in [1, %d]", kMaxGroups);
  FERRY_CHECK_ARG(groups * n <= (int64_t)1 << 36, "bad sizes: groups * n above 2^36");
  FERRY_CHECK_ARG(starts || groups == 1, "starts must name the rows of several groups");
  return 0;
}

}  // namespace
}  // namespace lin
}  // namespace ferry

using namespace ferry;
using namespace ferry::lin;

extern "C" int64_t ferry_linear_workspace_bytes(int32_t op, int64_t pairs, int64_t n, int64_t k, int64_t groups) {
  if (pairs < 0 || pairs >= kMost || n < 1 || n >= kMost || k < 1 || k >= kMost || groups < 1 || groups > kMaxGroups)
    return -1;
  if (op == FERRY_LINEAR_GRAD_Z) {
    const int64_t s = slope_splits(pairs, groups);
    return s > 1 ? s * groups * n * 4 : 0;
  }
  if (op < kFwd || op > kDw) return -1;
  return part_bytes(op, plan(op, pairs, n, k, groups), pairs, n, k, groups);
}

extern "C" int ferry_expert_linear(const void* x, int32_t dtype, int64_t x_rows, int64_t k, int64_t x_stride,
                                   const int64_t* rows, int64_t pairs, const int64_t* starts, int64_t groups,
                                   const void* w, int64_t n, int64_t w_stride, int64_t w_group_stride,
                                   const void* bias, int64_t bias_stride, int32_t activation, const void* residual,
                                   int64_t residual_stride, void* pre, void* out, int64_t out_stride,
                                   int32_t zero_rest, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_sizes(dtype, pairs, n, k, groups, starts)) return rc;
  FERRY_CHECK_ARG(activation >= kNone && activation <= kGeluTanh, "unknown activation");
  FERRY_CHECK_ARG(x_rows >= 0 && (rows || x_rows >= pairs), "x must have a row for every output row");
  FERRY_CHECK_ARG((x_stride >= k || x_rows <= 1) && (w_stride >= k || n == 1) && (out_stride >= n || pairs <= 1) && w_group_stride >= 0 &&
                      bias_stride >= 0 && (!residual || residual_stride >= 0),
                  "strides must reach over their rows");
  if (pairs == 0) return 0;
  FERRY_CHECK_ARG((x || x_rows == 0) && w && out, "null pointer argument");
  Args a = {};
  a.a = (const uint16_t*)x, a.lda = row_stride(x_stride, x_rows, k);
  a.b = (const uint16_t*)w, a.ldb = row_stride(w_stride, n, k), a.b_group = w_group_stride;
  a.out = (uint16_t*)out, a.ldo = row_stride(out_stride, pairs, n);
  a.starts = starts, a.rows = rows, a.x_rows = x_rows;
  a.J = n, a.C = k, a.groups = (int32_t)groups;
  a.act = activation, a.zero_rest = starts && zero_rest;
  a.bias = (const uint16_t*)bias, a.bias_group = bias_stride;
  a.residual = (const uint16_t*)residual, a.ldr = row_stride(residual_stride, pairs, n);
  a.pre = (uint16_t*)pre;
  return run<kFwd>(a, dtype, pairs, n, k, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int ferry_linear_grad_z(const void* grad, int32_t dtype, int64_t pairs, int64_t n, int64_t grad_stride,
                                   const void* pre, int32_t activation, const int64_t* starts, int64_t groups, void* dz,
                                   void* db, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_sizes(dtype, pairs, n, 1, groups, starts)) return rc;
  FERRY_CHECK_ARG(activation >= kNone && activation <= kGeluTanh, "unknown activation");
  FERRY_CHECK_ARG(grad_stride >= n || pairs <= 1, "strides must reach over their rows");
  FERRY_CHECK_ARG(activation == kNone || pairs == 0 || (pre && dz), "pre and dz belong to an activation");
  FERRY_CHECK_ARG(!starts || activation == kNone, "groups have no activation");
  if (activation == kNone && !db) return 0;
  FERRY_CHECK_ARG(pairs == 0 || grad, "null pointer argument");
  SlopeArgs a = {};
  a.splits = (int32_t)slope_splits(pairs, groups);
  const int64_t need = db && a.splits > 1 ? a.splits * groups * n * 4 : 0;
  FERRY_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), "workspace too small (%lld < %lld bytes)",
                  (long long)workspace_bytes, (long long)need);
  FERRY_CHECK_ARG(need == 0 || (uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
  a.dy = (const uint16_t*)grad, a.pre = (const uint16_t*)pre, a.dz = (uint16_t*)dz, a.db = (uint16_t*)db;
  a.part = (float*)workspace, a.ldy = grad_stride, a.pairs = pairs, a.N = n;
  a.starts = starts, a.groups = (int32_t)groups, a.act = activation;
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel, int cols) {
    launch("linear_slope", kernel, dim3((unsigned)std::min<int64_t>(ceil_div(n, cols) * groups * a.splits, kMaxGrid)), dim3(256), 0, s, a);
  };
  const bool few = ceil_div(n, 64) * groups < 128;
  if (dtype == FERRY_BF16)
    a.splits > 1 ? go(slope_kernel<Bf16, 8>, 256) : (few ? go(slope_kernel<Bf16, 128>, 16) : go(slope_kernel<Bf16, 32>, 64));
  else
    a.splits > 1 ? go(slope_kernel<F16, 8>, 256) : (few ? go(slope_kernel<F16, 128>, 16) : go(slope_kernel<F16, 32>, 64));
  FERRY_LAUNCHED("linear_slope");
  if (need) {
    const dim3 g2((unsigned)std::min<int64_t>(ceil_div(groups * n, 64), 65536));
    if (dtype == FERRY_BF16)
      launch("linear_slope_join", slope_join_kernel<Bf16>, g2, dim3(256), 0, s, (const float*)a.part, groups * n, (int)a.splits, a.db);
    else
      launch("linear_slope_join", slope_join_kernel<F16>, g2, dim3(256), 0, s, (const float*)a.part, groups * n, (int)a.splits, a.db);
    FERRY_LAUNCHED("linear_slope_join");
  }
  return 0;
}

extern "C" int ferry_expert_linear_grad_x(const void* dz, int32_t dtype, int64_t pairs, int64_t n, int64_t dz_stride,
                                          const int64_t* starts, int64_t groups, const void* w, int64_t k,
                                          int64_t w_stride, int64_t w_group_stride, void* out, int32_t zero_rest,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_sizes(dtype, pairs, n, k, groups, starts)) return rc;
  FERRY_CHECK_ARG((dz_stride >= n || pairs <= 1) && (w_stride >= k || n == 1) && w_group_stride >= 0,
                  "strides must reach over their rows");
  if (pairs == 0) return 0;
  FERRY_CHECK_ARG(dz && w && out, "null pointer argument");
  Args a = {};
  a.a = (const uint16_t*)dz, a.lda = row_stride(dz_stride, pairs, n);
  a.b = (const uint16_t*)w, a.ldb = row_stride(w_stride, n, k), a.b_group = w_group_stride;
  a.out = (uint16_t*)out, a.ldo = k;
  a.starts = starts, a.J = k, a.C = n, a.groups = (int32_t)groups, a.zero_rest = starts && zero_rest;
  return run<kDx>(a, dtype, pairs, n, k, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int ferry_expert_linear_grad_w(const void* dz, int32_t dtype, int64_t pairs, int64_t n, int64_t dz_stride,
                                          const void* x, int64_t x_rows, int64_t k, int64_t x_stride,
                                          const int64_t* rows, const int64_t* starts, int64_t groups, void* dw,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_sizes(dtype, pairs, n, k, groups, starts)) return rc;
  FERRY_CHECK_ARG(x_rows >= 0 && (rows || x_rows >= pairs), "x must have a row for every row of the gradient");
  FERRY_CHECK_ARG((dz_stride >= n || pairs <= 1) && (x_stride >= k || x_rows <= 1), "strides must reach over their rows");
  FERRY_CHECK_ARG(dw && (pairs == 0 || (dz && (x || x_rows == 0))), "null pointer argument");
  Args a = {};
  a.a = (const uint16_t*)dz, a.lda = row_stride(dz_stride, pairs, n);
  a.b = (const uint16_t*)x, a.ldb = row_stride(x_stride, x_rows, k);
  a.out = (uint16_t*)dw, a.ldo = k, a.o_group = n * k;
  a.starts = starts, a.rows = rows, a.x_rows = x_rows;
  a.I = n, a.J = k, a.groups = (int32_t)groups;
  return run<kDw>(a, dtype, pairs, n, k, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int ferry_sum_pairs(const void* part, int32_t dtype, int64_t pairs, int64_t k, const int32_t* pair_pos,
                               int64_t tokens, int64_t topk, void* out, void* stream) {
  clear_error();
  FERRY_CHECK_ARG(dtype == FERRY_BF16 || dtype == FERRY_F16, "dtype must be bf16 or fp16");
  FERRY_CHECK_ARG(pairs >= 0 && pairs < kMost && k >= 1 && k < kMost && tokens >= 0 && tokens < kMost && topk >= 1 && topk < kMost, "bad sizes");
  if (tokens == 0) return 0;
  FERRY_CHECK_ARG(out && pair_pos && (part || pairs == 0), "null pointer argument");
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(tokens * ceil_div(k, 8), 256), 1 << 20));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == FERRY_BF16)
    launch("sum_pairs", sum_pairs_kernel<Bf16>, grid, dim3(256), 0, s, (const uint16_t*)part, pairs, k, k, pair_pos, tokens, (int)topk, (uint16_t*)out);
  else
    launch("sum_pairs", sum_pairs_kernel<F16>, grid, dim3(256), 0, s, (const uint16_t*)part, pairs, k, k, pair_pos, tokens, (int)topk, (uint16_t*)out);
  FERRY_LAUNCHED("sum_pairs");
  return 0;
}
