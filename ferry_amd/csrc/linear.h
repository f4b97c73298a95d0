// What the kernels of the linear products share: their arguments, the groups' table of tiles, loads of
// 16-bit operands, the epilogue.
//
// Three products over G groups of rows, starts[g] <= p < starts[g + 1] (one group of all rows for a
// dense layer), with i the index of an output row, j that of an output column, c the contraction:
//   kFwd  y[p, j]  = sum_c x[row(p), c] w[g][j, c]     i = p, j < N, c < K
//   kDx   dx[p, j] = sum_c dz[p, c] w[g][c, j]         i = p, j < K, c < N
//   kDw   dw[g][i, j] = sum_p dz[p, i] x[row(p), j]    i < N, j < K, c = p
// Operand A belongs to i, B to j.  An operand whose elements follow each other along c (x and w in kFwd,
// dz in kDx) is staged in LDS by rows of its own index; the others (w in kDx, both of kDw) by rows of c,
// and their fragments are read with the transposing LDS read, so that no operand is copied in another
// order first.
#pragma once

#include "common.h"

namespace ferry {
namespace lin {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

enum { kFwd = 0, kDx = 1, kDw = 2 };
enum { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3, kGeluTanh = 4 };   // FERRY_ACT_*

constexpr int kMaxGroups = FERRY_MAX_EXPERTS;

struct Args {
  const uint16_t* a;    // x (kFwd), dz (kDx, kDw)
  const uint16_t* b;    // w (kFwd, kDx), x (kDw)
  int64_t lda, ldb, ldo;           // elements from row to row
  int64_t b_group, o_group;        // elements from group to group: weights, dw
  const int64_t* starts;           // null: one group of all pairs
  const int64_t* rows;             // null: row(p) = p
  int64_t pairs, x_rows;           // rows of the grouped order, rows of x
  int64_t I, J, C;                 // sizes of i, j and c; the ragged one is 0
  int32_t groups, splits;          // parts of the contraction, joined by join_kernel
  int32_t act, zero_rest;          // zero_rest: rows outside the groups become 0
  int32_t vec_out;                 // out, residual and pre take 8-byte accesses of four columns
  int64_t bias_group;
  const uint16_t* bias;
  const uint16_t* residual;
  int64_t ldr;
  uint16_t* pre;
  uint16_t* out;
  float* part;                     // [splits][rows of out][J], with splits > 1
};

// -- types -------------------------------------------------------------------------------------

struct Bf16 {
  static constexpr int32_t kType = FERRY_BF16;
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mma(s16x8 p, s16x8 q, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, p), __builtin_bit_cast(x8, q), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float load(uint16_t h) { return bf16_to_f32(h); }
  static __device__ __forceinline__ uint16_t round(float f) { return f32_to_bf16(f); }
  static __device__ __forceinline__ uint32_t round2(float lo, float hi) {   // lo | hi << 16
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, b16x2));
  }
};
struct F16 {
  static constexpr int32_t kType = FERRY_F16;
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mma(s16x8 p, s16x8 q, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, p), __builtin_bit_cast(x8, q), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float load(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }
  static __device__ __forceinline__ uint16_t round(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
  static __device__ __forceinline__ uint32_t round2(float lo, float hi) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, h16x2));
  }
};

// -- activations ---------------------------------------------------------------------------------
// fp32, with the hardware's exp2 and reciprocal: a relative error of about 1e-6, in the tails, where an exponential
// multiplies the rounding of its argument, of up to 2e-5 (the results are rounded to 8 or 11 bits afterwards).  The
// tanh form is z / (1 + e^-2u), u = sqrt(2 / pi) (z + 0.044715 z^3): no cancellation for negative z.

// 1 / (1 + 2^-y): two transcendental instructions, which cost as much as eight others
__device__ __forceinline__ float sigmoid2(float y) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-y));
}
__device__ __forceinline__ float sigmoid(float z) { return sigmoid2(1.44269504f * z); }
// sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3), in powers of 2
__device__ __forceinline__ float gelu_gate(float z) { return sigmoid2(z * fmaf(0.102943240f, z * z, 2.30220819f)); }

// The normal distribution function, erfc(-z / sqrt 2) / 2, with erfc(x) = t e^(P(t) - x^2), t = 1 / (1 + x / 2), for x >= 0,
// the form that Press et al., Numerical Recipes, use.  P is a Chebyshev fit of degree 9 over 0 <= x <= 12 of our own to
// ln(erfc(x) e^(x^2) / t).  The fit's relative error is 6e-8; evaluated in fp32 the result's is 4e-7 for |z| < 1, 4e-6 up to 6
// and 1.7e-5 up to 12 (x's and x^2's roundings, times e^), where rounding to bf16 costs 4e-3; from about |z| = 13 on the
// result is 0.  An absolute error of 1e-7 would take fewer instructions, but gelu's tail would be lost.
__device__ __forceinline__ float normal_cdf(float z) {
  const float x = fabsf(z) * 0.70710678f, t = __builtin_amdgcn_rcpf(fmaf(0.5f, x, 1.0f));
  float p = 0.157751014f;
  p = fmaf(p, t, -0.750181579f);
  p = fmaf(p, t, 1.31865295f);
  p = fmaf(p, t, -0.909740677f);
  p = fmaf(p, t, 0.0943214298f);
  p = fmaf(p, t, -0.0902556599f);
  p = fmaf(p, t, 0.0652326513f);
  p = fmaf(p, t, 0.380354122f);
  p = fmaf(p, t, 0.999348078f);
  p = fmaf(p, t, -1.26548227f);
  const float q = 0.5f * t * __builtin_amdgcn_exp2f(1.44269504f * fmaf(-x, x, p));
  return z > 0.f ? 1.0f - q : q;
}

__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case kRelu: return z <= 0.f ? 0.f : z;   // a NaN stays one
    case kSilu: return z * sigmoid(z);
    case kGelu: return z * normal_cdf(z);
    case kGeluTanh: return z * gelu_gate(z);
    default: return z;
  }
}

// f'(z).  Beyond |z| = 30 those of gelu are 0 or 1 to all bits; the clamp keeps z^3 finite.  That of silu is beyond 200, and
// an infinite z, which a finite argument above fp16's largest is rounded to, would make 0 times infinity of it.
__device__ __forceinline__ float slope(int act, float z) {
  if (z != z) return z;
  switch (act) {
    case kRelu: return z <= 0.f ? 0.f : 1.f;
    case kSilu: {
      z = fminf(fmaxf(z, -200.f), 200.f);
      const float s = sigmoid(z);
      return s * (1.0f + z * (1.0f - s));
    }
    case kGelu: {
      z = fminf(fmaxf(z, -30.f), 30.f);
      return normal_cdf(z) + z * 0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * z * z);
    }
    case kGeluTanh: {
      z = fminf(fmaxf(z, -30.f), 30.f);
      const float s = gelu_gate(z);
      return s + z * s * (1.0f - s) * 1.5957691f * (1.0f + 0.134145f * z * z);
    }
    default: return 1.f;
  }
}

// -- groups ----------------------------------------------------------------------------------------

// The rows of group g are [start, start + n), forced into [0, pairs], so that whatever starts holds every
// access stays inside the tensors; a group that ends before it starts has none.
__device__ __forceinline__ int in_pairs(const Args& a, int64_t s) { return (int)(s < 0 ? 0 : (s > a.pairs ? a.pairs : s)); }
__device__ __forceinline__ int group_start(const Args& a, int g) { return in_pairs(a, a.starts[g]); }

struct Table {
  __attribute__((aligned(16))) int32_t cum[kMaxGroups];   // tiles before the group, 0x7fffffff behind the last
  int32_t rows[kMaxGroups];
  uint16_t order[kMaxGroups];   // not RAGGED_I: the groups by descending rows
  int32_t total, first, last;   // tiles; rows of the grouped order before the first and behind the last group
};

// The groups' rows and tiles: `rows` rows a tile with RAGGED_I, else `rows` tiles for each group, whose order is by
// descending rows.  start (nullable): the groups' first rows.  Loads and sums by wavefront 0, all loads at once.
template <bool RAGGED_I>
__device__ __forceinline__ void build_table(const Args& a, Table& t, int rows, int32_t* start = nullptr) {
  constexpr int Q = kMaxGroups / 64;
  const int G = a.groups;
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int64_t lo[Q] = {}, hi[Q] = {};
    int64_t end = a.pairs, begin = 0;
    if (a.starts) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (q * 64 < G) {
          const int g = q * 64 + lane < G ? q * 64 + lane : G - 1;
          lo[q] = a.starts[g];
          hi[q] = a.starts[g + 1];
        }
      begin = a.starts[0];
      end = a.starts[G];
    } else {
      hi[0] = a.pairs;
    }
    int sum = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int g = q * 64 + lane;
      if (q * 64 < G) {
        const int s = in_pairs(a, lo[q]), e = in_pairs(a, hi[q]), n = e > s && g < G ? e - s : 0;
        const int c = g < G ? (RAGGED_I ? (int)(((uint32_t)n + rows - 1) / (uint32_t)rows) : rows) : 0;
        int incl = c;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const int v = __shfl_up(incl, off, 64);
          if (lane >= off) incl += v;
        }
        t.cum[g] = g < G ? sum + incl - c : 0x7fffffff;
        if (start) start[g] = s;
        t.rows[g] = n;
        sum += __shfl(incl, 63, 64);
      } else {
        t.cum[g] = 0x7fffffff;
      }
    }
    if (lane == 0) {
      t.total = sum;
      t.first = in_pairs(a, begin);
      t.last = in_pairs(a, end);
    }
  }
  __syncthreads();
  if constexpr (!RAGGED_I) {
    for (int g = threadIdx.x; g < G; g += blockDim.x) {
      const int n = t.rows[g];
      int rank = 0;
      for (int h = 0; h < G; ++h) rank += t.rows[h] > n || (t.rows[h] == n && h < g);
      t.order[rank] = (uint16_t)g;
    }
    __syncthreads();
  }
}

// the group of tile m: the last g with cum[g] <= m (groups without tiles share their successor's)
__device__ __forceinline__ int find_group(const Table& t, int m) {
  const int lane = threadIdx.x & 63;
  int le = 0;
#pragma unroll
  for (int q = 0; q < kMaxGroups / 256; ++q) {
    const u32x4 c = *reinterpret_cast<const u32x4*>(&t.cum[(q * 64 + lane) * 4]);
#pragma unroll
    for (int k = 0; k < 4; ++k) le += __popcll(__ballot((int)c[k] <= m));
  }
  return __builtin_amdgcn_readfirstlane(le - 1);
}

// -- operands in LDS ---------------------------------------------------------------------------------
// Rows of 16-byte chunks, chunk c of row r in place c ^ swizzle(r).
// By index ("direct"): 64 values of c a row (128 bytes); a fragment is 16 rows by one chunk, lane l of the
// wavefront row l % 16, chunk l / 16 of the step's four: the 16 rows of a quarter wavefront then lie on
// 16 different chunks of the banks.
// By c ("across"): W indices a row.  The transposing read takes from each of 16 lanes 8 bytes, lanes
// 4 r + q four indices 4 q of the row c = r, and gives lane l the index l at four c: two of them make a
// fragment, lane group g the c = 8 g .. 8 g + 7.  32 lanes read 8 rows (4 of each group) of 32 bytes,
// which the swizzle puts on 64 different banks.
__device__ __forceinline__ int swz_direct(int r) { return (r >> 1) & 7; }
template <int W>
__device__ __forceinline__ int swz_across(int r) {
  if (W == 32) return ((r >> 3) & 1) << 1;
  return W == 64 ? ((((r >> 1) & 1) | (((r >> 3) & 1) << 1)) << 1) : (((r & 3) | (((r >> 3) & 1) << 2)) << 1);
}
// fragment of 16 indices from i0 on at K step ks (32 values of c): byte offsets into the staged operand
__device__ __forceinline__ uint32_t frag_direct(int i0, int ks) {
  const int lane = threadIdx.x & 63, r = i0 + (lane & 15);
  return (uint32_t)(r * 128 + (((4 * ks + (lane >> 4)) ^ swz_direct(r)) << 4));
}
template <int W>
__device__ __forceinline__ uint32_t frag_across(int i0, int ks, int h) {
  const int lane = threadIdx.x & 63, r = (lane & 15) >> 2, q = lane & 3;
  const int c = 32 * ks + 8 * (lane >> 4) + 4 * h + r;
  const int i = i0 + 4 * q;
  return (uint32_t)(c * W * 2 + ((((i >> 3)) ^ swz_across<W>(c)) << 4) + (i & 4) * 2);
}
typedef __attribute__((address_space(3))) const s16x8 lds_x8;
typedef __attribute__((address_space(3))) s16x4 lds_x4;
__device__ __forceinline__ s16x8 read_direct(uint32_t addr) { return *reinterpret_cast<lds_x8*>((uintptr_t)addr); }
__device__ __forceinline__ s16x8 read_across(uint32_t lo, uint32_t hi) {
  const s16x4 p = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_x4*>((uintptr_t)lo));
  const s16x4 q = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_x4*>((uintptr_t)hi));
  return s16x8{p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
}

// -- epilogue ----------------------------------------------------------------------------------------
// Four columns j .. j + 3 (of which `n` > 0 are there) of output row `row`: bias, pre, activation,
// residual, one rounding.  g: the group, for its bias.
template <typename T>
__device__ __forceinline__ void finish4(const Args& a, int g, int64_t row, int64_t j, int n, f32x4 v) {
  uint16_t* const o = a.out + row * a.ldo + j;
  const bool whole = n >= 4 && a.vec_out;
  if (a.bias) {
    const uint16_t* b = a.bias + g * a.bias_group + j;
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] += q < n ? T::load(b[q]) : 0.f;
  }
  if (a.pre) {
    uint16_t* const p = a.pre + row * a.J + j;
    if (whole) {
      *reinterpret_cast<u32x2*>(p) = u32x2{T::round2(v[0], v[1]), T::round2(v[2], v[3])};
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q < n) p[q] = T::round(v[q]);
    }
  }
  if (a.act != kNone) {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = activate(a.act, v[q]);
  }
  if (a.residual) {
    const uint16_t* r = a.residual + row * a.ldr + j;
    if (whole) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(r);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += T::load((uint16_t)(w[q >> 1] >> (16 * (q & 1))));
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q < n) v[q] += T::load(r[q]);
    }
  }
  if (whole) {
    *reinterpret_cast<u32x2*>(o) = u32x2{T::round2(v[0], v[1]), T::round2(v[2], v[3])};
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < n) o[q] = T::round(v[q]);
  }
}

// rows of the output before the first and behind the last group, by all workgroups of a launch
__device__ __forceinline__ void zero_rest(const Args& a, int first, int last) {
  const int64_t n = first + (a.pairs - last);
  for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
    uint16_t* const o = a.out + (r < first ? r : last + (r - first)) * a.ldo;
    for (int64_t j = threadIdx.x; j < a.J; j += blockDim.x) o[j] = 0;
  }
}

}  // namespace lin
}  // namespace ferry
