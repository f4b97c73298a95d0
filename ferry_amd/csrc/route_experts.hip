// Expert selection of a general gate: scores s = softmax(logits) or 1 / (1 + e^-logits), choice scores
// c = s + bias, expert groups scored by their largest c or by the sum of their two largest, the
// best topk_groups groups, of those the k experts with the largest c, weights s of the chosen ones
// (renormalised, scaled, rounded to bf16).  Ties go to the lowest index, of groups and of experts.
//
// No counterpart in the reference, whose gates are softmax + top-k (ferry/model.py:141-157) in torch's
// CPU order; router.hip serves those.
//
// Scores, sums and comparisons are 64-bit: two experts whose scores differ by less than an fp32
// step are told apart, so the selection is that of the formulas and does not hang on a kernel's
// rounding.  The card's fp64 rate is its fp32 rate, so this costs registers and not time.
//
// A choice score that is a NaN counts as -infinity, as do experts with a logit of -infinity
// (masked experts, also where a bias is added): such experts are chosen last, and their weights are what
// the formulas give (0 for a masked one).  The chosen IDs are always k distinct ones in [0, E).
#include "common.h"

namespace ferry {
namespace {

constexpr int kMaxRouteExperts = 512;
constexpr int kWaves = 4;

struct RouteArgs {
  const void* logits;
  const float* bias;   // [E] or null
  int64_t tokens;
  int32_t experts, topk, groups, topk_groups;
  int32_t sigmoid, top2, renorm;
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

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v = fmax(v, __shfl_xor(v, off, 64));
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v = min(v, __shfl_xor(v, off, 64));
  return v;
}

// orders a wavefront's LDS accesses (its lanes run in step: no wait is needed)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// One wavefront per token; lane l holds the experts l + 64 j.  An expert that cannot be chosen (any
// more) has a NaN for its choice score: fmax and comparisons pass it over.
template <typename T, int N>
__global__ __launch_bounds__(64 * kWaves) void route_experts_kernel(RouteArgs a) {
  __shared__ double choice[kWaves][64 * N];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double kInf = __builtin_huge_val();
  for (int64_t t = (int64_t)blockIdx.x * kWaves + wave; t < a.tokens; t += (int64_t)gridDim.x * kWaves) {
    double s[N], c[N];
    double top = -kInf, sum = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = lane + 64 * j;
      s[j] = e < a.experts ? load_logit<T>(a.logits, t * a.experts + e) : -kInf;
      top = fmax(top, s[j]);
    }
    if (!a.sigmoid) top = wave_max(top);
    // softmax: an infinite or NaN logit makes every weight of the row a NaN (a row of masked experts
    // alone: 0)
    bool nan = false;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const double x = s[j];
      if (a.sigmoid) {
        s[j] = 1.0 / (1.0 + exp(-x));
      } else {
        s[j] = x == -kInf ? 0.0 : exp(x - top);
        sum += s[j];
      }
      c[j] = x == -kInf ? -kInf : 0.0;
    }
    if (!a.sigmoid) {
      sum = wave_sum(sum);
      nan = sum != sum;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = lane + 64 * j;
      if (!a.sigmoid) s[j] = nan ? __builtin_nan("") : (sum > 0 ? s[j] / sum : 0.0);
      if (e < a.experts) {
        const double v = s[j] + (a.bias ? (double)a.bias[e] : 0.0);
        c[j] = c[j] == -kInf || v != v ? -kInf : v;
      } else {
        c[j] = __builtin_nan("");
      }
    }
    if (a.groups > 1) {
#pragma unroll
      for (int j = 0; j < N; ++j) choice[wave][lane + 64 * j] = c[j];
      wave_sync();
      const int size = a.experts / a.groups;
      double mine[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int g = lane + 64 * j;
        mine[j] = -kInf;
        if (g < a.groups) {
          double b1 = -kInf, b2 = -kInf;
          for (int i = 0; i < size; ++i) {
            const double v = choice[wave][g * size + i];
            b2 = fmax(b2, fmin(b1, v));
            b1 = fmax(b1, v);
          }
          mine[j] = a.top2 ? b1 + b2 : b1;
          if (mine[j] != mine[j]) mine[j] = -kInf;   // +inf and -inf biases in one group
        }
      }
      wave_sync();
#pragma unroll
      for (int j = 0; j < N; ++j) choice[wave][lane + 64 * j] = mine[j];
      wave_sync();
      // an expert stays open if fewer than topk_groups groups beat its own
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int e = lane + 64 * j, g = e / size;
        if (e < a.experts) {
          const double own = choice[wave][g];
          int better = 0;
          for (int o = 0; o < a.groups; ++o) {
            const double v = choice[wave][o];
            better += v > own || (v == own && o < g);
          }
          if (better >= a.topk_groups) c[j] = __builtin_nan("");
        }
      }
      wave_sync();
    }
    // k rounds: the largest choice score, the lowest expert that has it
    double total = 0, wk = 0;
    int ek = 0;   // lane j keeps the j-th chosen expert
    for (int r = 0; r < a.topk; ++r) {
      double m = c[0];
#pragma unroll
      for (int j = 1; j < N; ++j) m = fmax(m, c[j]);
      m = wave_max(m);
      int e = 0x7fffffff;
#pragma unroll
      for (int j = N - 1; j >= 0; --j)
        if (c[j] == m) e = lane + 64 * j;
      e = wave_min(e);
      double w = 0;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (e == lane + 64 * j) {
          w = s[j];
          c[j] = __builtin_nan("");
        }
      w = __shfl(w, e & 63, 64);
      total += w;
      if (lane == r) wk = w, ek = e;
    }
    if (lane < a.topk) {
      if (a.renorm) wk = total > 0 || total != total ? wk / total : 0.0;
      a.idx[t * a.topk + lane] = ek;
      a.w[t * a.topk + lane] = f32_to_bf16((float)(wk * (double)a.scale));
    }
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
  a.tokens = tokens;
  a.experts = (int32_t)experts;
  a.topk = (int32_t)topk;
  a.groups = (int32_t)groups;
  a.topk_groups = (int32_t)topk_groups;
  a.sigmoid = sigmoid != 0;
  a.top2 = group_top2 != 0;
  a.renorm = renorm != 0;
  a.scale = scale;
  a.idx = idx_out;
  a.w = (bf16_t*)w_out_bf16;
  const int64_t wgs = ceil_div(tokens, kWaves);
  const dim3 grid((unsigned)(wgs < kMaxGrid ? wgs : kMaxGrid)), block(64 * kWaves);
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto t) {
    typedef decltype(t) T;
    if (experts <= 64) launch("route_experts", route_experts_kernel<T, 1>, grid, block, 0, s, a);
    else if (experts <= 128) launch("route_experts", route_experts_kernel<T, 2>, grid, block, 0, s, a);
    else if (experts <= 256) launch("route_experts", route_experts_kernel<T, 4>, grid, block, 0, s, a);
    else launch("route_experts", route_experts_kernel<T, 8>, grid, block, 0, s, a);
  };
  if (dtype == FERRY_BF16) go(bf16_t{});
  else if (dtype == FERRY_F32) go(float{});
  else go((_Float16)0);
  FERRY_LAUNCHED("route_experts");
  return 0;
}
