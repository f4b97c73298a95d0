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
  int row0, rows, j0;    // output row of the tile's first, rows from there on (may be more than a tile's), first column
  int p0;                // pair of the tile's first row (kFwd) or c (kDw)
};

// The tiles that a workgroup takes: one of each round of gridDim.x of them.  Workgroup b runs on XCD b % 8; in a
// round those of one XCD take a contiguous run.  kDw's groups come by descending rows, and so their tiles by
// descending time: every other round runs backwards, so that who had the longest tile of one round gets the
// shortest of the next (65,536 rows of 128 experts by a Zipf law, 1,536 x 2,048: 757 -> 706 us).  The others'
// tiles stay in the groups' order: a group's partial tile then shares w in L2 with its whole ones, which is worth
// more than rounds of equal tiles (y of the same: 530 us; partial tiles last 560, spread evenly between whole ones
// 546).
// A tile's place takes several divisions and a search; 16 lanes find those of 16 rounds at once and leave them in
// LDS, where a wavefront reads what it needs.  Each wavefront does so for itself, all writing the same, which
// needs no barrier; two sets in turn, since they are not all at the same place.
constexpr int kRun = 16;
template <int MODE, bool GATHER, int TM, int TN>
struct Tiles {
  static constexpr bool XA = MODE == kDw, XB = MODE != kFwd, RAG = MODE != kDw;
  struct Entry {
    u32x4 a, b, c;   // a and b: address, size and nc, rows (0: no such tile); c: row0, j0, g | s << 16, p0
  };
  struct Store {
    __attribute__((aligned(16))) Entry e[2 * kRun];
  };
  const Args& args;
  const Table& tt;
  Entry* e;
  int rounds, at;

  __device__ __forceinline__ Tiles(const Args& args, const Table& tt, Store& store) : args(args), tt(tt), e(store.e), at(-1) {
    const int grid = (int)gridDim.x, ntj = (int)ceil_div(args.J, TN);
    rounds = (tt.total * ntj * args.splits + grid - 1) / grid;
    rounds = __builtin_amdgcn_readfirstlane(rounds);
  }

  // the places of rounds k .. k + 15
  __device__ __forceinline__ void fill(int k0) {
    const int lane = threadIdx.x & 63;
    if (lane >= kRun) return;
    const Args& a = args;
    const int grid = (int)gridDim.x, ntj = (int)ceil_div(a.J, TN), nti = RAG ? 0 : (int)ceil_div(a.I, TM);
    const int items = tt.total * ntj * a.splits, k = k0 + lane;
    const bool xcds = grid % 8 == 0;
    const int slot = xcds ? (int)(blockIdx.x % 8) * (grid / 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x;
    const int item = k * grid + (!RAG && (k & 1) ? grid - 1 - slot : slot);
    Entry out = {};
    if (item < items) {
      const int s = item % a.splits, q = item / a.splits;
      int mt, jt, i0, g;
      // bands of four row tiles, all columns of a band before the next: what runs at one time on an XCD shares
      // few rows of either operand
      auto banded = [&](int n, int rows) __attribute__((always_inline)) {
        const int band = n / (4 * ntj), r = n - band * 4 * ntj, h = rows - 4 * band < 4 ? rows - 4 * band : 4;
        jt = r / h;
        mt = 4 * band + r - jt * h;
      };
      if constexpr (RAG) {
        banded(q, tt.total);
        g = 0;   // the last group whose cum is at most mt (groups without tiles share their successor's)
#pragma unroll
        for (int step = kMaxGroups / 2; step; step >>= 1)
          if (g + step < a.groups && tt.cum[g + step] <= mt) g += step;
        i0 = (mt - tt.cum[g]) * TM;
      } else {
        const int rank = q / (nti * ntj);
        banded(q - rank * nti * ntj, nti);
        g = tt.order[rank];
        i0 = mt * TM;
      }
      const int64_t start = a.starts ? group_start(a, g) : 0;
      const int n = tt.rows[g], rows = (RAG ? n : (int)a.I) - i0, j0 = jt * TN;
      const int C = RAG ? (int)a.C : n, per = ((C + a.splits - 1) / a.splits + 63) & ~63;
      const int c0 = s * per, nc = C - c0 < per ? (C > c0 ? C - c0 : 0) : per;
      const int64_t row0 = (RAG ? start : 0) + i0, vi = rows < TM ? rows : TM, vj = a.J - j0 < TN ? a.J - j0 : TN;
      auto buffer = [&](const uint16_t* p, int64_t rows, int64_t ld, int64_t last) __attribute__((always_inline)) {
        const int64_t size = rows > 0 && last > 0 ? ((rows - 1) * ld + last) * 2 : 0;
        return u32x4{(uint32_t)(uintptr_t)p, (uint32_t)((uint64_t)(uintptr_t)p >> 32) & 0xffffu,
                     (uint32_t)(size > 0xffffffffll ? 0xffffffffll : size), 0u};
      };
      if constexpr (XA)
        out.a = buffer(a.a + (start + c0) * a.lda + i0, nc, a.lda, vi);
      else if constexpr (GATHER && MODE == kFwd)
        out.a = buffer(a.a + c0, a.x_rows, a.lda, nc);
      else
        out.a = buffer(a.a + row0 * a.lda + c0, vi, a.lda, nc);
      const uint16_t* const w = a.b + (MODE == kDw ? 0 : g * a.b_group);
      if constexpr (!XB)
        out.b = buffer(w + (int64_t)j0 * a.ldb + c0, vj, a.ldb, nc);
      else if constexpr (GATHER && MODE == kDw)
        out.b = buffer(w + j0, a.x_rows, a.ldb, vj);
      else
        out.b = buffer(w + ((MODE == kDw ? start : 0) + c0) * a.ldb + j0, nc, a.ldb, vj);
      out.a[3] = nc;
      out.b[3] = rows;
      out.c = u32x4{(uint32_t)row0, (uint32_t)j0, (uint32_t)(g | s << 16), (uint32_t)(MODE == kFwd ? row0 : start + c0)};
    }
    e[(k0 & kRun) + lane] = out;
  }
  // the next round with a tile for this workgroup; false behind the last
  __device__ __forceinline__ bool next() {
    while (++at < rounds) {
      if (at % kRun == 0) fill(at);
      if (__builtin_amdgcn_readfirstlane((int)e[at % (2 * kRun)].b[3])) return true;
    }
    return false;
  }
  // the tile of the present round
  __device__ __forceinline__ Tile tile() const {
    const Entry& r = e[at % (2 * kRun)];
    const u32x4 qa = r.a, qb = r.b, qc = r.c;
    auto s = [](uint32_t v) __attribute__((always_inline)) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    Tile t;
    t.a = u32x4{s(qa[0]), s(qa[1]), s(qa[2]), 0x00020000u};
    t.b = u32x4{s(qb[0]), s(qb[1]), s(qb[2]), 0x00020000u};
    t.nc = (int)s(qa[3]);
    t.rows = (int)s(qb[3]);
    t.row0 = (int)s(qc[0]);
    t.j0 = (int)s(qc[1]);
    t.g = (int)(s(qc[2]) & 0xffffu);
    t.s = (int)(s(qc[2]) >> 16);
    t.p0 = (int)s(qc[3]);
    return t;
  }
};

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
// the choice of the activation once for eight
__device__ __forceinline__ void activate8(int act, float (&v)[8]) {
  auto all = [&](auto a) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = activate(decltype(a)::value, v[q]);
  };
  switch (act) {
    case kRelu: return all(std::integral_constant<int, kRelu>{});
    case kSilu: return all(std::integral_constant<int, kSilu>{});
    case kGelu: return all(std::integral_constant<int, kGelu>{});
    default: return all(std::integral_constant<int, kGeluTanh>{});
  }
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

// dw is stored past the caches (non-temporal), whose lines the operands keep: a training step of 3,000 rows of 64
// experts, 2,048 x 1,408, 318 -> 300 us; of 65,536 rows of 128 experts and of one dense layer the same time.  y and dx,
// whose readers come at once, are not: they gain or lose 1 %.
constexpr int kPast = 2;

// The epilogue of a tile: eight consecutive columns of a row at a time, through buffers that begin at the tile's
// first row and column and end with its last row, so that rows behind it are dropped without a test and an address
// is one 32-bit offset; columns behind the last lie nowhere.
template <typename T, int MODE, int TM, int TN>
struct Output {
  __amdgpu_buffer_rsrc_t out, pre, res;
  uint32_t ldo, ldp, ldr;   // bytes from row to row
  int32_t act;
  bool parts, keep;

  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)(uint32_t)bytes, 0x00020000);
  }
  __device__ __forceinline__ Output(const Args& a, const Tile& t) : act(a.act), parts(a.splits > 1), keep(a.pre != nullptr) {
    const int64_t rows = t.rows < TM ? t.rows : TM, cols = a.J - t.j0 < TN ? a.J - t.j0 : TN, row0 = t.row0;
    if (parts) {
      const int64_t at = MODE != kDw ? t.s * a.pairs + row0 : ((int64_t)t.s * a.groups + t.g) * a.I + row0;
      out = buffer(a.part + at * a.J + t.j0, ((rows - 1) * a.J + cols) * 4);
      ldo = (uint32_t)a.J * 4;
    } else {
      const uint16_t* const o = a.out + (MODE == kDw ? t.g * a.o_group : 0);
      out = buffer(o + row0 * a.ldo + t.j0, ((rows - 1) * a.ldo + cols) * 2);
      ldo = (uint32_t)a.ldo * 2;
    }
    if constexpr (MODE == kFwd) {
      pre = buffer(a.pre + row0 * a.J + t.j0, ((rows - 1) * a.J + cols) * 2);
      res = buffer(a.residual + row0 * a.ldr + t.j0, ((rows - 1) * a.ldr + cols) * 2);
      ldp = (uint32_t)a.J * 2;
      ldr = (uint32_t)a.ldr * 2;
    }
  }
  // the residual of row r (bytes r * ldr + 2 j), 0 behind the tile's end
  __device__ __forceinline__ u32x4 residual(uint32_t at) const { return __builtin_amdgcn_raw_buffer_load_b128(res, at, 0, 0); }
  // v + bias, pre, activation (ACT -1: the call's), residual r, one rounding; or the sums of a part.  ro and rp: the
  // row's offsets in out and pre, j: the first column in the tile, `in`: whether it is there
  template <int ACT>
  __device__ __forceinline__ void store(uint32_t ro, uint32_t rp, int j, bool in, float (&v)[8], const u32x4& bias,
                                        const u32x4& r) const {
    if (parts) {
      const uint32_t at = in ? ro + j * 4 : kNowhere - 16;
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}), out, at, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]}), out, at, 16, 0);
      return;
    }
    float f[8];
    if constexpr (MODE == kFwd) {
      unpack8<T>(bias, f);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += f[q];
    }
    if constexpr (ACT != kNone) {
      if (keep) __builtin_amdgcn_raw_buffer_store_b128(pack8<T>(v), pre, in ? rp + j * 2 : kNowhere, 0, 0);
      if constexpr (ACT > 0) {
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = activate(ACT, v[q]);
      } else if (act != kNone) {
        activate8(act, v);
      }
    }
    if constexpr (MODE == kFwd) {
      unpack8<T>(r, f);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += f[q];
    }
    __builtin_amdgcn_raw_buffer_store_b128(pack8<T>(v), out, in ? ro + j * 2 : kNowhere, 0, MODE == kDw ? kPast : 0);
  }
};

}  // namespace
}  // namespace lin
}  // namespace ferry
