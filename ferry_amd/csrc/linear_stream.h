// What the tiled kernels of the linear products share: where a tile lies, and its epilogue.
#pragma once

#include "linear_loads.h"

namespace ferry {
namespace lin {
namespace {

// LDS places of the rows of a direct B operand: a fragment takes the rows 8 g + 4 c + [0, 4), g < 4
__device__ __forceinline__ int swz_pair(int r) { return ((r >> 1) & 1) | (((r >> 3) & 3) << 1); }

struct Tile {
  u32x4 a, b;            // the operands as buffers that end with the tile's rows, columns and contraction
  int g, s, nc;          // group, part, length of the contraction
  int64_t row0;          // output row of the tile's first
  int rows, j0;          // rows from there on (may be more than a tile's), first column
  const int64_t* idx;    // row numbers from the tile's first row (kFwd) or c (kDw) on
};

// The tiles that a workgroup takes: one of each round of gridDim.x.  Workgroup b runs on XCD b % 8; in a round
// those of one XCD take a contiguous run.  kDw's groups come by descending rows, whose tiles take as long as
// these are many, so every other round runs backwards: who had the longest tile of one round gets the shortest
// of the next.  (65,536 rows of 128 experts by a Zipf law of exponent 1.1, 1,536 x 2,048: in the groups' order
// 757 us.)
struct Rounds {
  int slot, round, total;
  bool snake;
  __device__ __forceinline__ Rounds(int total, bool snake) : round(0), total(total), snake(snake) {
    const int per_xcd = gridDim.x % 8 == 0 ? (int)gridDim.x / 8 : 0;
    slot = per_xcd ? (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8) : (int)blockIdx.x;
  }
  __device__ __forceinline__ int at(int r) const {   // the tile of round r, or one that is not there
    return r * (int)gridDim.x + (snake && (r & 1) ? (int)gridDim.x - 1 - slot : slot);
  }
};

// The tile `item`.  Bands of four row tiles, all columns of a band before the next: what runs at one time on
// an XCD shares few rows of either operand.  mtiles: of all groups; nti: of a group in kDw.
template <int MODE, bool GATHER, int TM, int TN>
__device__ __forceinline__ Tile locate_tile(const Args& a, const Table& tt, int item, int mtiles, int nti, int ntj) {
  constexpr bool XA = MODE == kDw, XB = MODE != kFwd, RAG = MODE != kDw;
  Tile t;
  t.s = item % a.splits;
  const int q = item / a.splits;
  int mt, jt, i0;
  auto banded = [&](int k, int rows) __attribute__((always_inline)) {
    const int band = k / (4 * ntj), r = k - band * 4 * ntj, h = rows - 4 * band < 4 ? rows - 4 * band : 4;
    jt = r / h;
    mt = 4 * band + r - jt * h;
  };
  if constexpr (RAG) {
    banded(q, mtiles);
    t.g = a.starts ? find_group(tt, mt) : 0;
    i0 = (mt - tt.cum[t.g]) * TM;
  } else {
    const int rank = q / (nti * ntj);
    banded(q - rank * nti * ntj, nti);
    t.g = tt.order[rank];
    i0 = mt * TM;
  }
  t.g = __builtin_amdgcn_readfirstlane(t.g);
  const int64_t start = tt.start[t.g], n = tt.rows[t.g];
  t.rows = __builtin_amdgcn_readfirstlane((int)((RAG ? n : a.I) - i0));
  t.j0 = __builtin_amdgcn_readfirstlane(jt * TN);
  t.row0 = (RAG ? start : 0) + i0;
  const int64_t C = RAG ? a.C : n, per = ceil_div(ceil_div(C, a.splits), 64) * 64;
  const int64_t c0 = t.s * per, c1 = c0 + per < C ? c0 + per : C;
  t.nc = __builtin_amdgcn_readfirstlane((int)(c1 > c0 ? c1 - c0 : 0));
  const int64_t nc = t.nc, vi = t.rows < TM ? t.rows : TM, vj = a.J - t.j0 < TN ? a.J - t.j0 : TN;
  auto size = [](int64_t rows, int64_t ld, int64_t last) { return rows > 0 && last > 0 ? ((rows - 1) * ld + last) * 2 : 0; };
  if constexpr (XA)
    t.a = buffer_at(a.a + (start + c0) * a.lda + i0, size(nc, a.lda, vi));
  else if constexpr (GATHER && MODE == kFwd)
    t.a = buffer_at(a.a + c0, size(a.x_rows, a.lda, nc));
  else
    t.a = buffer_at(a.a + t.row0 * a.lda + c0, size(vi, a.lda, nc));
  const uint16_t* const w = a.b + (MODE == kDw ? 0 : t.g * a.b_group);
  if constexpr (!XB)
    t.b = buffer_at(w + (int64_t)t.j0 * a.ldb + c0, size(vj, a.ldb, nc));
  else if constexpr (GATHER && MODE == kDw)
    t.b = buffer_at(w + t.j0, size(a.x_rows, a.ldb, vj));
  else
    t.b = buffer_at(w + ((MODE == kDw ? start : 0) + c0) * a.ldb + t.j0, size(nc, a.ldb, vj));
  t.idx = GATHER ? a.rows + (MODE == kFwd ? t.row0 : start + c0) : nullptr;
  return t;
}

template <typename T>
__device__ __forceinline__ void unpack8(const u32x4& v, float (&f)[8]) {
#pragma unroll
  for (int q = 0; q < 8; ++q) f[q] = T::load((uint16_t)(v[q >> 1] >> (16 * (q & 1))));
}
template <typename T>
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  u32x4 w;
#pragma unroll
  for (int q = 0; q < 4; ++q) w[q] = T::round2(f[2 * q], f[2 * q + 1]);
  return w;
}
// columns j .. j + 7 of row `row`: v + bias, pre, activation (ACT -1: the call's), residual r, one rounding
template <typename T, int ACT>
__device__ __forceinline__ void finish8(const Args& a, uint16_t* out, int64_t row, int64_t j, float (&v)[8],
                                        const u32x4& bias, const u32x4& r) {
  float f[8];
  unpack8<T>(bias, f);
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] += f[q];
  if constexpr (ACT != kNone) {
    if (a.pre) *reinterpret_cast<u32x4*>(a.pre + row * a.J + j) = pack8<T>(v);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = activate(ACT < 0 ? a.act : ACT, v[q]);
  }
  unpack8<T>(r, f);
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] += f[q];
  *reinterpret_cast<u32x4*>(out + row * a.ldo + j) = pack8<T>(v);
}

// Eight consecutive columns of a row from two tiles' accumulators.  Interleaved fragments (direct B) give
// 8 g + [0, 8) for the lanes' group g as they are; tiles of 16 consecutive columns (ACROSS) exchange their odd
// and even groups, and give 16 (g % 2) + 8 (g / 2) + [0, 8).  By all lanes.
template <bool ACROSS>
__device__ __forceinline__ void columns8(const f32x4& t0, const f32x4& t1, float (&v)[8]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float lo = t0[q], hi = t1[q];
    if constexpr (ACROSS) {
      const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(lo), __float_as_uint(hi), false, false);
      lo = __uint_as_float(s[0]);
      hi = __uint_as_float(s[1]);
    }
    v[q] = lo;
    v[4 + q] = hi;
  }
}

// columns j .. j + 7 of the tile's row r: the output, or the sums of a part of the contraction
template <typename T, int MODE, int ACT>
__device__ __forceinline__ void store8(const Args& a, const Tile& t, uint16_t* out, int r, int64_t j, float (&v)[8],
                                       const u32x4& bias, const u32x4& res) {
  const int64_t row = t.row0 + r;
  if (a.splits > 1) {
    float* const o = a.part + (MODE != kDw ? t.s * a.pairs + row : ((int64_t)t.s * a.groups + t.g) * a.I + row) * a.J + j;
    *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    finish8<T, ACT>(a, out, row, j, v, bias, res);
  }
}

}  // namespace
}  // namespace lin
}  // namespace ferry
