// Expert selection of a general gate: scores s = softmax(logits) or 1 / (1 + e^-logits), choice scores
// c = s + bias, expert groups scored by their largest c or by the sum of their two largest, the
// best topk_groups groups, of those the k experts with the largest c, weights s of the chosen ones
// (renormalised, scaled, rounded to bf16).  Ties go to the lowest index, of groups and of experts.
//
// No counterpart in the reference, whose gates are softmax + top-k (ferry/model.py:141-157) in torch's
// CPU order; router.hip serves those.
//
// Scores, sums and comparisons are 64-bit: two experts whose scores differ by less than an fp32 step are told
// apart, so the selection is that of the formulas and does not hang on a kernel's rounding.
//
// A choice score that is a NaN counts as -infinity, as do experts with a logit of -infinity
// (masked experts, also where a bias is added): such experts are chosen last, and their weights are what
// the formulas give (0 for a masked one).  The chosen IDs are always k distinct ones in [0, E).
//
// Small calls are bound by the latency of one token's chain, and a wavefront takes a token (exact_row).  Large ones
// are bound by instruction issue, and 16 lanes take one, every step serving four.  They need 64 bits for few
// experts only: fp32 scores, which are within a known margin of the true ones, tell which can be
// among the k best.  These are drawn by 32-bit keys, the high bits of the score over the expert's
// index (unique: a drawing needs no second search for its owner), until the key is below the k-th's by more than
// the margin.  The candidates, one to a lane, are ranked by their 64-bit scores.  A row with more than 16 of
// them, or whose group scores are too near each other for fp32, goes to exact_row.  One token of 256 experts in 8
// groups, top 8: 6.2 us; 32,768 of them, fp32: 29 us (27 a call where calls follow each other), against 105 with a
// wavefront a token and 7 for the bytes at the rate of a large copy; what is left is instructions (1,220 vector and 320
// scalar ones for four tokens, 16 us of issue) and, at the end, the last rows of exact_row (about 6 us).  An eighth
// wavefront on a SIMD changes nothing.  Batches of more than 256 experts or more than 16 chosen have a wavefront a token too:
// 32,768 tokens, 512 experts in 8 groups 104 us (bytes 13), 256 experts and 24 of them 87 (bytes 8).
//
// The margin.  e^y as 2^(y log2 e) in fp32 is off by at most (2.5 |y| + 2) 2^-24 of itself: y's and the product's
// rounding, the constant's and the instruction's.  Without a bias an expert's choice score is 1 / (1 + e^-x) or
// e^(x - max) alone (the sum does not change a row's order): above 2^-100, |y| <= 70, two of them are off by less
// than 2^-15 together, below that by less than 2^-98.  With a bias it is s + bias: s is off by less than 2^-21
// (s (1 - s) |x| < 0.23 for a sigmoid, e^-y y < 0.37 for a softmax, whose sum is a 64-bit one), the addition by
// 2^-24 of its result.  So 2^-14 of the score and 2^-98, with a bias 2^-20 of it and 2^-18, cover two experts; and
// two groups' two each, if "the score" is the largest among them.
#include "common.h"

#include <type_traits>

namespace ferry {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kMaxRouteExperts = 512;
constexpr int kWaves = 4;
constexpr int64_t kLaunchRows = 1 << 24;   // a grid has less than 2^32 threads
// Tokens up to which a whole wavefront takes one.  256 experts in 8 groups: 9.4 us against 9.2 with 16 lanes at 2,048
// tokens, 12.9 against 13.7 at 4,096; 128 experts without groups: 5.8 against 5.6 and 8.4 against 5.5.
constexpr int64_t kWide = 2048;

struct RouteArgs {
  const void* logits;
  const float* bias;   // [E] or null
  int64_t first, tokens;   // of this launch: [first, tokens)
  int32_t experts, topk, groups, topk_groups;
  int32_t top2, renorm;
  float scale;
  int64_t* idx;
  bf16_t* w;
};

template <typename T>
__device__ __forceinline__ double load_logit(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 4) return (double)((const float*)p)[i];
  else if constexpr (__is_same(T, bf16_t)) return (double)bf16_to_f32(((const bf16_t*)p)[i]);
  else return (double)(float)((const _Float16*)p)[i];
}

// e^x to about 1e-14: 2^n times the Taylor polynomial of e^(f ln 2), |f| <= 1/2, of degree 11 (next term
// 0.3466^12 / 12! = 6e-15).  x below -800 gives 0, above 800 infinity, NaN a NaN.
__device__ __forceinline__ double exp64(double x) {
  const double y = fmin(fmax(x, -800.0), 800.0) * 1.4426950408889634074;
  const double n = __builtin_rint(y), f = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = __builtin_fma(p, f, 1.0 / 3628800.0);
  p = __builtin_fma(p, f, 1.0 / 362880.0);
  p = __builtin_fma(p, f, 1.0 / 40320.0);
  p = __builtin_fma(p, f, 1.0 / 5040.0);
  p = __builtin_fma(p, f, 1.0 / 720.0);
  p = __builtin_fma(p, f, 1.0 / 120.0);
  p = __builtin_fma(p, f, 1.0 / 24.0);
  p = __builtin_fma(p, f, 1.0 / 6.0);
  p = __builtin_fma(p, f, 0.5);
  p = __builtin_fma(p, f, 1.0);
  p = __builtin_fma(p, f, 1.0);
  p = __builtin_amdgcn_ldexp(p, (int)n);
  return x != x ? x : p;
}
// 1 / d for d >= 1: the hardware's estimate and two Newton steps; infinity gives 0
__device__ __forceinline__ double rcp64(double d) {
  double r = __builtin_amdgcn_rcp(d);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  return d == __builtin_huge_val() ? 0.0 : r;
}
__device__ __forceinline__ double sigmoid64(double x) { return rcp64(1.0 + exp64(-x)); }

// a value of another lane of the same 16, and reductions over them, which every lane gets
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, ((uint64_t)dpp<CTRL>((uint32_t)(u >> 32)) << 32) | dpp<CTRL>((uint32_t)u));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kRor1 = 0x121;
template <typename F>
__device__ __forceinline__ double reduce16(double v, F f) {
  v = f(v, dpp64<kXor1>(v));
  v = f(v, dpp64<kXor2>(v));
  v = f(v, dpp64<kHalfMirror>(v));
  return f(v, dpp64<kMirror>(v));
}
template <typename F>
__device__ __forceinline__ float reduce16(float v, F f) {
  auto u = [](float x) { return __float_as_uint(x); };
  v = f(v, __uint_as_float(dpp<kXor1>(u(v))));
  v = f(v, __uint_as_float(dpp<kXor2>(u(v))));
  v = f(v, __uint_as_float(dpp<kHalfMirror>(u(v))));
  return f(v, __uint_as_float(dpp<kMirror>(u(v))));
}
__device__ __forceinline__ uint32_t largest16(uint32_t v) {
  v = max(v, dpp<kXor1>(v));
  v = max(v, dpp<kXor2>(v));
  v = max(v, dpp<kHalfMirror>(v));
  return max(v, dpp<kMirror>(v));
}
// over a wavefront
template <typename F>
__device__ __forceinline__ double reduce64(double v, F f) {
  v = reduce16(v, f);
  auto of = [&](int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane) << 32) |
                                          (uint32_t)__builtin_amdgcn_readlane((int)u, lane));
  };
  return f(f(of(0), of(16)), f(of(32), of(48)));
}
struct Sum {
  template <typename X>
  __device__ __forceinline__ X operator()(X a, X b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ double operator()(double a, double b) const { return fmax(a, b); }
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
// keeps the two largest of b1 >= b2 and v
template <typename X>
__device__ __forceinline__ void keep_two(X& b1, X& b2, X v) {
  b2 = Max()(b2, v < b1 ? v : b1);
  b1 = Max()(b1, v);
}
// Batcher's odd-even merge sort, descending
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int d = p; d >= 1; d /= 2)
#pragma unroll
      for (int j = d % p; j + d < N; j += 2 * d)
#pragma unroll
        for (int i = 0; i < d; ++i)
          if (i + j + d < N && (i + j) / (2 * p) == (i + j + d) / (2 * p)) {
            const uint32_t hi = max(k[i + j], k[i + j + d]), lo = min(k[i + j], k[i + j + d]);
            k[i + j] = hi;
            k[i + j + d] = lo;
          }
}
// orders a wavefront's LDS accesses (its lanes run in step: no wait is needed)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// weight of a chosen expert's score
__device__ __forceinline__ bf16_t weight_of(const RouteArgs& a, double s, double total) {
  if (a.renorm) s = total > 0 || total != total ? s / total : 0.0;
  return f32_to_bf16((float)(s * (double)a.scale));
}

// the choice score of a logit x with score s
__device__ __forceinline__ double choice_of(const RouteArgs& a, double x, double s, int e) {
  const double v = s + (a.bias ? (double)a.bias[e] : 0.0);
  return x == -__builtin_huge_val() || v != v ? -__builtin_huge_val() : v;
}

// The score of a logit, of a row with the given largest logit (NaNs aside) and 1 / sum: a softmax is 0 for a masked
// expert, a NaN in a row with a NaN or an infinity, 0 in a row of masked experts alone.
__device__ __forceinline__ double softmax_exp(double x, double top) {
  return x == -__builtin_huge_val() ? 0.0 : exp64(x - top);
}
template <bool SIGMOID>
__device__ __forceinline__ double score_of(double x, double top, double inv) {
  if constexpr (SIGMOID) return sigmoid64(x);
  else return softmax_exp(x, top) * inv;
}
__device__ __forceinline__ double inverse_sum(double sum) { return sum > 0 ? 1.0 / sum : sum; }

// Row t by a wavefront, 64-bit throughout; lane l holds the experts l + 64 j.  lds: 64 N + groups doubles and as many
// words as groups.  Experts that cannot be chosen have a NaN, which fmax and comparisons pass over.
template <typename T, bool SIGMOID, int N>
__device__ __forceinline__ void exact_row(const RouteArgs& a, int64_t t, double* lds) {
  const double kInf = __builtin_huge_val(), kNan = __builtin_nan("");
  const int lane = threadIdx.x & 63;
  double x[N], c[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = lane + 64 * j;
    x[j] = e < a.experts ? load_logit<T>(a.logits, t * a.experts + e) : -kInf;
  }
  double top = -kInf, inv = 0;
  if constexpr (!SIGMOID) {
    double sum = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) top = fmax(top, x[j]);
    top = reduce64(top, Max());
#pragma unroll
    for (int j = 0; j < N; ++j) sum += softmax_exp(x[j], top);
    inv = inverse_sum(reduce64(sum, Sum()));
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = lane + 64 * j;
    c[j] = e < a.experts ? choice_of(a, x[j], score_of<SIGMOID>(x[j], top, inv), e) : kNan;
  }
  if (a.groups > 1) {
    const int size = a.experts / a.groups;
    double* const groups = lds + 64 * N;
    int32_t* const open = (int32_t*)(groups + a.groups);
#pragma unroll
    for (int j = 0; j < N; ++j) lds[lane + 64 * j] = c[j];
    wave_sync();
    for (int g = lane; g < a.groups; g += 64) {
      double b1 = -kInf, b2 = -kInf;
#pragma unroll 4
      for (int i = 0; i < size; ++i) keep_two(b1, b2, lds[g * size + i]);
      const double v = a.top2 ? b1 + b2 : b1;
      groups[g] = v != v ? -kInf : v;   // +inf and -inf biases in one group
    }
    wave_sync();
    // a group stays open if fewer than topk_groups groups beat it
    for (int g = lane; g < a.groups; g += 64) {
      const double own = groups[g];
      int better = 0;
#pragma unroll 4
      for (int o = 0; o < a.groups; ++o) {
        const double v = groups[o];
        better += v > own || (v == own && o < g);
      }
      open[g] = better < a.topk_groups;
    }
    wave_sync();
    const float per = 1.0f / (float)size;   // a group's number: exact below 2^20 experts with the half added
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = lane + 64 * j;
      if (e < a.experts && !open[(int)(((float)e + 0.5f) * per)]) c[j] = kNan;
    }
    wave_sync();
  }
  int mine = 0;   // lane j: the j-th chosen expert
  for (int r = 0; r < a.topk; ++r) {
    double m = c[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = fmax(m, c[j]);
    m = reduce64(m, Max());
    int e = 0;
#pragma unroll
    for (int j = N - 1; j >= 0; --j) {
      const uint64_t at = __ballot(c[j] == m);
      if (at) e = 64 * j + __ffsll((unsigned long long)at) - 1;
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (e == lane + 64 * j) c[j] = kNan;
    if (lane == r) mine = e;
  }
  double s = 0;
  if (lane < a.topk) s = score_of<SIGMOID>(load_logit<T>(a.logits, t * a.experts + mine), top, inv);
  const double total = reduce64(s, Sum());
  if (lane < a.topk) {
    a.idx[t * a.topk + lane] = mine;
    a.w[t * a.topk + lane] = weight_of(a, s, total);
  }
}

template <typename T, bool SIGMOID, int N>
__global__ __launch_bounds__(64 * kWaves) void route_wide(RouteArgs a) {
  extern __shared__ double lds[];
  const int wave = threadIdx.x >> 6;
  double* const own = lds + wave * (64 * N + a.groups + (a.groups + 1) / 2);
  const int64_t t = a.first + (int64_t)blockIdx.x * kWaves + wave;
  if (t < a.tokens) exact_row<T, SIGMOID, N>(a, t, own);
}

// The logits (or biases) of four consecutive experts, those past the last -infinity.  Rows begin at any multiple of
// an element.
template <typename T>
__device__ __forceinline__ void load_quad(const T* row, int e, int experts, float* x) {
  const T* const p = row + e;
  T v[4];
  if (e + 4 <= experts) {
    __builtin_memcpy(v, p, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p[e + i < experts ? i : -e];   // the row's first one
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f;
    if constexpr (__is_same(T, bf16_t)) f = bf16_to_f32(v[i]);
    else f = (float)v[i];
    x[i] = e + i < experts ? f : -__builtin_huge_valf();
  }
}

__device__ __forceinline__ float margin_of(const RouteArgs& a, float v) {
  return a.bias ? fabsf(v) * 0x1p-20f + 0x1p-18f : fabsf(v) * 0x1p-14f + 0x1p-98f;
}
// an fp32 number as an integer of the same order
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o ^ ((uint32_t)((int)~o >> 31) | 0x80000000u));
}

// 16 lanes a token; lane l of them holds the experts from 64 i + 4 l on, four for each i.  k up to 16.
template <typename T, bool SIGMOID, int N>
__global__ __launch_bounds__(64 * kWaves) void route_many(RouteArgs a) {
  constexpr int E = 16 * N;                       // experts, rounded up
  constexpr uint32_t kLow = 2 * E - 1;            // a key's low bits: the index, and one that is always set
  constexpr float kInf = __builtin_huge_valf();
  constexpr int kExact = (E + 63) / 64;
  // a wavefront's: [4] x (E choice scores, or the two largest of each four; group scores; words of the groups);
  // exact_row has the same room
  extern __shared__ double lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % 16, q = lane / 16;
  float* const own = (float*)lds + wave * 4 * (E + 2 * a.groups);
  float* const scores = own + q * E;
  float* const groups = own + 4 * E + q * a.groups;
  int32_t* const open = (int32_t*)(own + 4 * (E + a.groups)) + q * a.groups;
  auto expert = [&](int j) { return (j >> 2) * 64 + 4 * l + (j & 3); };
  const int size = a.experts / a.groups;
  const bool by_four = size % 4 == 0;
  const float per = 1.0f / (float)size;   // a group's number: exact below 2^20 experts with the half added
  // without a bias and with renormalised weights a softmax's sum drops out
  const bool sum_free = !a.bias && a.renorm;
  const int64_t t0 = a.first + ((int64_t)blockIdx.x * kWaves + wave) * 4;
  if (t0 >= a.tokens) return;
  const bool live = t0 + q < a.tokens;
  const int64_t t = live ? t0 + q : a.tokens - 1;   // the last row again: nothing is stored
  bool exact = false;                               // the row goes to exact_row
  float x[N];
#pragma unroll
  for (int j = 0; j < N; j += 4) load_quad((const T*)a.logits + t * a.experts, expert(j), a.experts, x + j);
  float most = -kInf;
  double inv = 1.0;
  if constexpr (!SIGMOID) {
#pragma unroll
    for (int j = 0; j < N; ++j) most = fmaxf(most, x[j]);
    most = reduce16(most, Max());
    if (!sum_free) {
      double sum = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) sum += softmax_exp((double)x[j], (double)most);
      inv = inverse_sum(reduce16(sum, Sum()));
    }
    float sum = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float v = __builtin_amdgcn_exp2f((x[j] - most) * 1.44269504f);
      sum += v;
      x[j] = x[j] == -kInf ? -1.0f : v;   // masked
    }
    sum = reduce16(sum, Sum());
    exact = !(sum >= 1.0f);   // a NaN or an infinity among the logits, or masked experts alone
    if (a.bias) {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= (float)inv;
    }
  }
  uint32_t key[N];   // 0: cannot be chosen
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    float c[4], b[4];
    if (a.bias) load_quad(a.bias, expert(j), a.experts, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = expert(j + i);
      float s = x[j + i];
      bool none = !SIGMOID && s < 0;   // masked
      if constexpr (SIGMOID) {
        none = s == -kInf;
        s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s * -1.44269504f));
      }
      if (a.bias) s += b[i];
      c[i] = none || s != s ? -kInf : s;
      key[j + i] = e < a.experts ? (ordered(c[i]) & ~kLow) | (uint32_t)(E + (E - 1 - e)) : 0u;
    }
    if (a.groups > 1) {
      if (by_four) {
        float b1 = fmaxf(c[0], c[1]), b2 = fminf(c[0], c[1]);
        keep_two(b1, b2, c[2]);
        keep_two(b1, b2, c[3]);
        *(f32x2*)&scores[expert(j) / 2] = (f32x2){b1, b2};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) scores[expert(j + i)] = c[i];
      }
    }
  }
  if (a.groups > 1) {
    wave_sync();
    float most_of = 0;   // the largest of the groups' scores
    for (int g = l; g < a.groups; g += 16) {
      float b1 = -kInf, b2 = -kInf;
      if (by_four) {
#pragma unroll 4
        for (int i = 0; i < size / 4; ++i) {
          const f32x2 v = *(const f32x2*)&scores[(g * size + 4 * i) / 2];
          b2 = fmaxf(fmaxf(b2, v[1]), fminf(b1, v[0]));
          b1 = fmaxf(b1, v[0]);
        }
      } else {
#pragma unroll 4
        for (int i = 0; i < size; ++i) keep_two(b1, b2, scores[g * size + i]);
      }
      const float v = a.top2 ? b1 + b2 : b1;
      groups[g] = v != v ? -kInf : v;
      const float m1 = fabsf(b1), m2 = a.top2 ? fabsf(b2) : 0;
      most_of = fmaxf(most_of, fmaxf(m1 < kInf ? m1 : 0, m2 < kInf ? m2 : 0));
    }
    most_of = reduce16(most_of, Max());
    wave_sync();
    // the last group that stays open and the first that does not have to be apart
    float last = -kInf, next = -kInf;
    for (int g = l; g < a.groups; g += 16) {
      const float mine = groups[g];
      int better = 0;
#pragma unroll 4
      for (int o = 0; o < a.groups; ++o) {
        const float v = groups[o];
        better += v > mine || (v == mine && o < g);
      }
      open[g] = better < a.topk_groups;
      if (better == a.topk_groups - 1) last = mine;
      if (better == a.topk_groups) next = mine;
    }
    last = reduce16(last, Max());
    next = reduce16(next, Max());
    exact = exact || !(last - next > margin_of(a, most_of));
    wave_sync();
    if (by_four) {   // four experts at once are of one group
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const int e = expert(j);
        const bool can = e < a.experts && open[(int)(((float)e + 0.5f) * per)];
#pragma unroll
        for (int i = 0; i < 4; ++i) key[j + i] = can ? key[j + i] : 0u;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int e = expert(j);
        if (e < a.experts && !open[(int)(((float)e + 0.5f) * per)]) key[j] = 0u;
      }
    }
  }
  // Each lane sorts its keys; a drawing takes the largest of the lanes' first ones.  The r-th goes to lane r.
  sort_keys(key);
  uint32_t mine = 0, m = 0;
  auto draw = [&](int r) {
    if (l == r) mine = m;
    const bool owner = key[0] == m;   // its keys move up
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint32_t up = j + 1 < N ? key[j + 1] : 0u;
      const uint32_t stay = key[j];   // values, not places: a chosen place would become a search through all keys
      key[j] = owner ? up : stay;
    }
  };
  for (int r = 0; r < a.topk; ++r) {
    m = largest16(key[0]);
    draw(r);
  }
  const float kth = unordered(m & ~kLow);
  const uint32_t floor = fabsf(kth) < 0x1p100f ? ordered(kth - margin_of(a, kth)) & ~kLow : 0u;
  bool more = !exact;
  for (int r = a.topk; r < 17; ++r) {
    m = largest16(key[0]);
    more = more && m != 0 && (m & ~kLow) >= floor;
    if (!__any(more)) break;
    if (more) {
      draw(r);
      exact = r == 16;
    }
  }
  const bool cand = mine != 0;
  const int e = cand ? E - 1 - (int)(mine & (E - 1)) : 0;
  const double logit = load_logit<T>(a.logits, t * a.experts + e);
  const double s = score_of<SIGMOID>(logit, (double)most, inv);
  const double v = cand ? choice_of(a, logit, s, e) : __builtin_nan("");
  // the r-th lane's is the r-th best, unless two near ones are the other way round
  double ov = dpp64<kRor1>(v);
  int oe = (int)dpp<kRor1>((uint32_t)e), ol = (int)dpp<kRor1>((uint32_t)l), rank = l;
  const bool ahead = ov > v || (ov == v && oe < e);
  if (__any(cand && ((ol == l - 1 && !ahead) || (ol == l + 1 && ahead)))) {
    rank = ahead;
#pragma unroll
    for (int i = 1; i < 15; ++i) {
      ov = dpp64<kRor1>(ov);
      oe = (int)dpp<kRor1>((uint32_t)oe);
      rank += ov > v || (ov == v && oe < e);
    }
  }
  const bool chosen = cand && rank < a.topk;
  const double total = reduce16(chosen ? s : 0.0, Sum());
  if (live && !exact && chosen) {
    a.idx[t * a.topk + rank] = e;
    a.w[t * a.topk + rank] = weight_of(a, s, total);
  }
  uint64_t rows = __ballot(exact && live && l == 0);
  wave_sync();
  while (rows) {
    const int64_t row = t0 + (__ffsll((unsigned long long)rows) - 1) / 16;
    rows &= rows - 1;
    exact_row<T, SIGMOID, kExact>(a, row, (double*)own);
    wave_sync();
  }
}

}  // namespace
}  // namespace ferry

using namespace ferry;

extern "C" int ferry_route_experts(const void* logits, int32_t dtype, int64_t tokens, int64_t experts,
                                   int64_t topk, int32_t sigmoid, const float* bias, int64_t groups,
                                   int64_t topk_groups, int32_t group_top2, int32_t renorm, float scale,
                                   int64_t* idx_out, void* w_out_bf16, void* stream) {
  clear_error();
  FERRY_CHECK_ARG(tokens >= 0, "bad sizes");
  FERRY_CHECK_ARG(experts >= 1 && experts <= kMaxRouteExperts, "experts must be in [1, %d]", kMaxRouteExperts);
  FERRY_CHECK_ARG(groups >= 1 && experts % groups == 0, "experts must be a multiple of groups");
  FERRY_CHECK_ARG(topk_groups >= 1 && topk_groups <= groups, "topk_groups must be in [1, groups]");
  FERRY_CHECK_ARG(topk >= 1 && topk <= 32 && topk <= topk_groups * (experts / groups),
                  "topk must be in [1, 32] and at most the experts of topk_groups groups");
  FERRY_CHECK_ARG(dtype == FERRY_BF16 || dtype == FERRY_F32 || dtype == FERRY_F16, "unknown dtype %d", dtype);
  FERRY_CHECK_ARG(!group_top2 || groups == 1 || experts / groups >= 2,
                  "a group's two largest scores need two experts a group");
  FERRY_CHECK_ARG(tokens < (int64_t)1 << 40, "too many tokens");
  if (tokens == 0) return 0;
  FERRY_CHECK_ARG(logits && idx_out && w_out_bf16, "null pointer argument");
  RouteArgs a;
  a.logits = logits;
  a.bias = bias;
  a.experts = (int32_t)experts;
  a.topk = (int32_t)topk;
  a.groups = topk_groups == groups ? 1 : (int32_t)groups;   // all stay open
  a.topk_groups = (int32_t)topk_groups;
  a.top2 = group_top2 != 0;
  a.renorm = renorm != 0;
  a.scale = scale;
  a.idx = idx_out;
  a.w = (bf16_t*)w_out_bf16;
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto t, auto sig, auto n) {
    constexpr int N = decltype(n)::value;   // 64 experts each
    const bool wide = tokens <= kWide || topk > 16 || N > 4;
    for (a.first = 0; a.first < tokens; a.first = a.tokens) {
      a.tokens = tokens - a.first < kLaunchRows ? tokens : a.first + kLaunchRows;
      const dim3 grid((unsigned)ceil_div(a.tokens - a.first, wide ? kWaves : 4 * kWaves));
      if (wide)
        launch("route_experts", route_wide<decltype(t), decltype(sig)::value, N>, grid, dim3(64 * kWaves),
               (uint32_t)(kWaves * 8 * (64 * N + a.groups + (a.groups + 1) / 2)), s, a);
      else if constexpr (N <= 4)
        launch("route_experts", route_many<decltype(t), decltype(sig)::value, 4 * N>, grid, dim3(64 * kWaves),
               (uint32_t)(kWaves * 16 * (64 * N + 2 * a.groups)), s, a);
    }
  };
  auto sized = [&](auto t, auto sig) {
    if (experts <= 64) go(t, sig, std::integral_constant<int, 1>{});
    else if (experts <= 128) go(t, sig, std::integral_constant<int, 2>{});
    else if (experts <= 256) go(t, sig, std::integral_constant<int, 4>{});
    else go(t, sig, std::integral_constant<int, 8>{});
  };
  auto typed = [&](auto t) {
    if (sigmoid) sized(t, std::true_type{});
    else sized(t, std::false_type{});
  };
  if (dtype == FERRY_BF16) typed(bf16_t{});
  else if (dtype == FERRY_F32) typed(float{});
  else typed((_Float16)0);
  FERRY_LAUNCHED("route_experts");
  return 0;
}
