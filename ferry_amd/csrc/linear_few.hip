// The linear products of few rows (a decode step, small batches): reading the weights is all they cost.
#include "linear_loads.h"
#include "linear_tile.h"

#include <algorithm>
#include <type_traits>

namespace ferry {
namespace lin {
namespace {

// A workgroup of WK wavefronts computes 16 MT rows by 16 NB columns; each wavefront takes every WK-th 64 of
// the contraction, and their sums are added through LDS, in wavefront order.  A wavefront streams the rows of
// w and x of its chunks through an LDS ring of its own, R chunks deep, by loads of whole 128-byte pieces of
// rows that are waited for one chunk at a time; no barrier stands in the loop.  Bound by reading w: rows of x
// that are not there cost nothing (they read as 0 without a transaction), the others come from L2.
// Workgroups stay and take items in turn (column blocks fastest), since a workgroup that finds no rows costs
// as much as its dispatch, and of 128 experts a decode step uses 40.
template <typename T, int MODE, bool GATHER, int MT, int NB, int WK, int R>
__global__ __launch_bounds__(64 * WK) void few_kernel(Args a) {
  constexpr bool XB = MODE == kDx;   // w staged by rows of the contraction
  constexpr int LW = 2 * NB, LX = 2 * MT, L = LW + LX, TN = 16 * NB;   // loads of a chunk; columns
  constexpr int kSlot = 16 * (NB + MT) * 128;
  static_assert(MT * NB * 1024 <= R * kSlot, "the sums of a wavefront fit its ring");
  __shared__ Table tt;
  __shared__ int32_t first_s[kMaxGroups];
  __shared__ __attribute__((aligned(1024))) char smem[WK * R * kSlot];
  __shared__ __attribute__((aligned(256))) uint32_t row_s[GATHER ? WK : 1][2][GATHER ? 64 : 1];
  if (a.starts) {
    build_table<true>(a, tt, 16 * MT, first_s);
    if (a.zero_rest) zero_rest(a, tt.first, tt.last);
  }
  const int ntj = (int)ceil_div(a.J, 16 * NB);
  const int mtiles = a.starts ? __builtin_amdgcn_readfirstlane(tt.total) : (int)ceil_div(a.pairs, 16 * MT);
  const int total = mtiles * ntj;
  const int tid = threadIdx.x, lane = tid & 63, r8 = lane >> 3;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t ring = lds_at(smem) + wave * R * kSlot;
  const uint32_t lda2 = (uint32_t)a.lda * 2, ldb2 = (uint32_t)a.ldb * 2;
  const int C = (int)a.C, steps = (C + 64 * WK - 1) / (64 * WK);
  for (int item = blockIdx.x; item < total; item += gridDim.x) {
    const int mt = item / ntj, j0 = (item - mt * ntj) * 16 * NB;
    int g = 0, start = 0, n = (int)a.pairs, m0 = mt * 16 * MT;
    if (a.starts) {
      g = find_group(tt, mt);
      m0 = (mt - __builtin_amdgcn_readfirstlane(tt.cum[g])) * 16 * MT;
      start = __builtin_amdgcn_readfirstlane(first_s[g]);
      n = __builtin_amdgcn_readfirstlane(tt.rows[g]);
    }
    const int vr = n - m0 < 16 * MT ? n - m0 : 16 * MT;   // rows, > 0
    const int64_t vj = a.J - j0 < 16 * NB ? a.J - j0 : 16 * NB;
    if constexpr (GATHER) {
      const u32x4 rows = buffer_at(a.rows + start + m0, (int64_t)vr * 8);
      load_lds4(rows, lane * 8, lds_at(row_s[wave][0]));
      load_lds4(rows, lane * 8 + 4, lds_at(row_s[wave][1]));
    }
    const u32x4 bw = XB ? buffer_at(a.b + g * a.b_group + j0, ((C - 1) * a.ldb + vj) * 2)
                        : buffer_at(a.b + g * a.b_group + (int64_t)j0 * a.ldb, ((vj - 1) * a.ldb + C) * 2);
    const u32x4 bx = GATHER ? buffer_at(a.a, ((a.x_rows - 1) * a.lda + C) * 2)
                            : buffer_at(a.a + (int64_t)(start + m0) * a.lda, ((vr - 1) * a.lda + C) * 2);
    uint32_t xo[LX];
    // chunk of place lane % 8 in the rows 8 q + lane / 8, and whether it lies in the contraction at step i
    auto chunk = [&](int q) __attribute__((always_inline)) { return (lane & 7) ^ swz_direct(8 * (q & 1) + r8); };
    auto load_w = [&](int i, int slot) __attribute__((always_inline)) {
      const int c = (i * WK + wave) * 64;
      const uint32_t dst = ring + slot * kSlot;
#pragma unroll
      for (int q = 0; q < LW; ++q) {
        if constexpr (XB) {
          const int r = 512 / TN * q + lane / (TN / 8), k = (lane % (TN / 8)) ^ swz_across<TN>(r);
          load_lds(bw, c < C ? (uint32_t)r * ldb2 + k * 16 : kNowhere, c < C ? c * ldb2 : 0, dst + 1024 * q);
        } else {
          load_lds(bw, c + chunk(q) * 8 < C ? (uint32_t)(8 * q + r8) * ldb2 + chunk(q) * 16 : kNowhere, c < C ? c * 2 : 0,
                   dst + 1024 * q);
        }
      }
    };
    auto load_x = [&](int i, int slot) __attribute__((always_inline)) {
      const int c = (i * WK + wave) * 64;
      const uint32_t dst = ring + slot * kSlot + LW * 1024;
#pragma unroll
      for (int q = 0; q < LX; ++q)
        load_lds(bx, c + chunk(q) * 8 < C ? xo[q] : kNowhere, c < C ? c * 2 : 0, dst + 1024 * q);
    };
#pragma unroll
    for (int i = 0; i < R; ++i) load_w(i, i);
    if constexpr (GATHER) wait_cnt<R * LW>();   // the row numbers, older than the weights
#pragma unroll
    for (int q = 0; q < LX; ++q) {
      const int r = 8 * q + r8;
      uint32_t x = r;
      bool ok = r < vr;
      if constexpr (GATHER) {
        x = row_s[wave][0][r];
        ok = ok && row_s[wave][1][r] == 0 && x < (uint64_t)a.x_rows;
      }
      xo[q] = ok ? x * lda2 + chunk(q) * 16 : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) load_x(i, i);
    f32x4 acc[MT][NB];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[i][b] = f32x4{0, 0, 0, 0};
    const int more = steps > R ? steps - R : 0;   // chunks that the loop loads
    auto step = [&](int i, int slot) __attribute__((always_inline)) {
      const uint32_t st = ring + slot * kSlot;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        s16x8 fw[NB], fx[MT];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          if constexpr (XB)
            fw[b] = read_across(st + frag_across<TN>(16 * b, ks, 0), st + frag_across<TN>(16 * b, ks, 1));
          else
            fw[b] = read_direct(st + frag_direct(16 * b, ks));
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) fx[m] = read_direct(st + LW * 1024 + frag_direct(16 * m, ks));
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[m][b] = T::mma(fw[b], fx[m], acc[m][b]);
      }
      if (i < more) {
        wait_lds();   // this chunk is read before its place is loaded anew
        load_w(i + R, slot);
        load_x(i + R, slot);
      }
    };
    // chunk i has landed when at most what was loaded after it is outstanding: of the first R, the rows of x
    // of the others and one chunk for each step so far; then the R - 1 chunks before it, or those left
    static_for<0, R>([&](auto ii) __attribute__((always_inline)) {
      constexpr int I = decltype(ii)::value;
      if (I < steps) {
        if (I <= more)
          wait_cnt<(R - 1 - I) * LX + I * L>();
        else
          wait_cnt<(R - 1 - I) * LX>();
        step(I, I);
      }
    });
    int slot = 0;
    for (int i = R; i < steps; ++i) {
      wait_chunks<R - 1, L>(steps - 1 - i);
      step(i, slot);
      slot = slot + 1 == R ? 0 : slot + 1;
    }
    wait_cnt<0>();
    // sums through LDS, over the rings
    __syncthreads();
    f32x4* const sums = reinterpret_cast<f32x4*>(smem);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int b = 0; b < NB; ++b) sums[(wave * MT * NB + m * NB + b) * 64 + lane] = acc[m][b];
    __syncthreads();
    for (int t = tid; t < MT * NB * 64; t += 64 * WK) {
      const int tile = t >> 6, l = t & 63, row = 16 * (tile / NB) + (l & 15), col = 16 * (tile % NB) + 4 * (l >> 4);
      f32x4 v = sums[tile * 64 + l];
#pragma unroll
      for (int w = 1; w < WK; ++w) v += sums[(w * MT * NB + tile) * 64 + l];
      const int m = (int)vj - col < 4 ? (int)vj - col : 4;
      if (row < vr && m > 0) finish4<T>(a, g, start + m0 + row, j0 + col, m, v);
    }
    __syncthreads();   // the rings are free again
  }
}

template <typename T, int MODE, bool GATHER>
void few_typed(int mt, int nb, const Args& a, int64_t tiles, int64_t cus, hipStream_t s) {
  const int64_t items = tiles * ceil_div(a.J, 16 * nb);
  auto go = [&](auto kernel, int threads, int resident) {
    launch("linear_few", kernel, dim3((unsigned)std::min(items, cus * resident)), dim3(threads), 0, s, a);
  };
  if constexpr (MODE == kFwd) {
    if (nb == 1 && items <= cus) return go(few_kernel<T, MODE, GATHER, 1, 1, 8, 4>, 512, 1);
    if (nb == 1) return go(few_kernel<T, MODE, GATHER, 1, 1, 4, 4>, 256, 2);
    if (mt == 1) return go(few_kernel<T, MODE, GATHER, 1, 2, 4, 3>, 256, 2);
  }
  if (mt == 2)
    go(few_kernel<T, MODE, GATHER, 2, 2, 4, 2>, 256, 2);
  else if (nb == 2)
    go(few_kernel<T, MODE, GATHER, 4, 2, 4, 2>, 256, 1);
  else
    go(few_kernel<T, MODE, GATHER, 4, 4, 4, 2>, 256, 1);
}
template <typename T>
void few_mode(int mode, int mt, int nb, const Args& a, int64_t tiles, int64_t cus, hipStream_t s) {
  if (mode == kDx) return few_typed<T, kDx, false>(mt, nb, a, tiles, cus, s);
  a.rows ? few_typed<T, kFwd, true>(mt, nb, a, tiles, cus, s) : few_typed<T, kFwd, false>(mt, nb, a, tiles, cus, s);
}

}  // namespace

void few_launch(int mode, int32_t dtype, int mt, int nb, const Args& a, int64_t tiles, int64_t cus, hipStream_t s) {
  dtype == FERRY_BF16 ? few_mode<Bf16>(mode, mt, nb, a, tiles, cus, s) : few_mode<F16>(mode, mt, nb, a, tiles, cus, s);
}

}  // namespace lin
}  // namespace ferry
