// MXFP4 rows: 4-bit elements (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one 8-bit
// power-of-two scale (2^(byte - 127), 255: NaN) per 32 consecutive elements of a row.
//
// Quantisation of a block: amax = max |x|, scale = 2^e with e = floor(log2(amax)) - 2 (6 = 1.5 * 2^2 is
// the largest element), at least 2^-127; each element is the e2m1 value nearest to x * 2^-e, ties to the
// even code, 6 above 5.  x * 2^-e is exact in fp32 wherever it can round to a non-zero element.
// A block that holds an infinity or a NaN has scale 255 and codes 0: it reads back as NaN.
// No counterpart in the reference, whose expert rows are bf16 only.
//
// Both directions are bound by memory: 294,912 rows of 2,048 bf16 elements are quantised in 305 us (5.0 TB/s read and
// written, a large copy's rate is 5.2) and read back in 317 us (4.8 TB/s).  Reading back writes four
// bytes for each one read: its stores bypass the caches (cached ones: 420 us, and 13.4 against 9.4 us for
// 4,096 x 4,096).  Two, four or eight loads of a lane in flight, and fewer workgroups that loop, were no faster.
#include "common.h"

#include <type_traits>

namespace ferry {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));   // any row's start

constexpr int kThreads = 256;
constexpr int kLaneElems = 8;   // elements of a lane: four lanes hold a block

// 8 elements of a row from column c0 on as fp32; columns past the last are 0.  Rows may begin at any
// multiple of the element size, so the full loads are unaligned ones.
template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same_v<T, bf16_t>) return bf16_to_f32(v);
  else return (float)v;
}
template <typename T>
__device__ __forceinline__ void load_elems(const T* row, int64_t c0, int64_t cols, float (&v)[8]) {
  T t[8];
  if (c0 + 8 <= cols) {
    __builtin_memcpy(t, row + c0, sizeof(t));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < cols ? to_float(row[c0 + i]) : 0.0f;
  }
}

// A workgroup takes kThreads consecutive lanes' work of the rows laid end to end (per lanes a row): one
// 64-bit division for the workgroup, a 32-bit one for each lane.
struct Place {
  int64_t row;
  uint32_t at;   // lane's place in the row
};
__device__ __forceinline__ Place place_of(int64_t first, uint32_t per) {
  const int64_t r0 = first / per;
  const uint32_t off = (uint32_t)(first - r0 * per) + threadIdx.x;
  const uint32_t dr = off / per;
  return {r0 + dr, off - dr * per};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void mxfp4_quantize_kernel(const T* __restrict__ x, int64_t ldx,
                                                                  int64_t cols, uint32_t per, int64_t total,
                                                                  uint8_t* __restrict__ codes, int64_t ldc,
                                                                  uint8_t* __restrict__ scales, int64_t lds) {
  for (int64_t first = (int64_t)blockIdx.x * kThreads; first < total; first += (int64_t)gridDim.x * kThreads) {
    if (first + threadIdx.x >= total) break;   // total is a multiple of 4: whole blocks leave together
    const Place p = place_of(first, per);
    float v[8];
    load_elems(x + p.row * ldx, (int64_t)p.at * kLaneElems, cols, v);
    uint32_t amax = 0;   // magnitudes compare like their bits; a NaN's are above all
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    amax = max(amax, (uint32_t)__builtin_amdgcn_mov_dpp((int)amax, 0xB1, 0xf, 0xf, true));   // lane ^ 1
    amax = max(amax, (uint32_t)__builtin_amdgcn_mov_dpp((int)amax, 0x4E, 0xf, 0xf, true));   // lane ^ 2
    const int ex = (int)(amax >> 23);            // biased exponent of amax
    const bool bad = ex == 255;
    const int byte = bad ? 255 : (ex > 2 ? ex - 2 : 0);
    const float inv = __uint_as_float((uint32_t)(bad ? 0 : 254 - byte) << 23);   // 2^(127 - byte)
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bad ? 0.0f : v[i] * inv;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], 1.0f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], 1.0f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], 1.0f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], 1.0f, 3);
    *(uint32_t*)(codes + p.row * ldc + (int64_t)p.at * 4) = c;
    if ((p.at & 3) == 0) scales[p.row * lds + (p.at >> 2)] = (uint8_t)byte;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes, int64_t ldc,
                                                                    const uint8_t* __restrict__ scales,
                                                                    int64_t lds, int64_t cols, uint32_t per,
                                                                    int64_t total, T* __restrict__ out,
                                                                    int64_t ldo) {
  for (int64_t first = (int64_t)blockIdx.x * kThreads; first < total; first += (int64_t)gridDim.x * kThreads) {
    if (first + threadIdx.x >= total) break;
    const Place p = place_of(first, per);
    const uint32_t c = *(const uint32_t*)(codes + p.row * ldc + (int64_t)p.at * 4);
    const uint32_t byte = scales[p.row * lds + (p.at >> 2)];
    // 2^(byte - 127) as fp32: 2^-127 is subnormal there
    const float s = __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255 ? 0x7fc00000u : byte << 23));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2);
    const f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    const float v[8] = {a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (std::is_same_v<T, bf16_t>) t[i] = f32_to_bf16(v[i] * s);
      else t[i] = (T)(v[i] * s);
    }
    const int64_t c0 = (int64_t)p.at * kLaneElems;
    T* const o = out + p.row * ldo + c0;
    if (c0 + 8 <= cols) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(t) / 16; ++i) {
        u32x4u w;
        __builtin_memcpy(&w, (const char*)t + 16 * i, 16);
        __builtin_nontemporal_store(w, (u32x4u*)o + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < cols) o[i] = t[i];
    }
  }
}

// the checks that both directions share; *empty: nothing to do
int check_rows(int64_t rows, int64_t cols, int64_t stride, int64_t ldc, int64_t lds, int32_t dtype,
               bool* empty) {
  const int64_t blocks = ceil_div(cols, 32);
  FERRY_CHECK_ARG(rows >= 0 && cols >= 0, "bad sizes");
  FERRY_CHECK_ARG(cols < ((int64_t)1 << 33) && rows < ((int64_t)1 << 48) / (cols + 32),
                  "rows of at most 2^33 elements, 2^48 in all");
  FERRY_CHECK_ARG(dtype == FERRY_BF16 || dtype == FERRY_F32 || dtype == FERRY_F16, "unknown dtype %d", dtype);
  *empty = rows == 0 || cols == 0;
  if (*empty) return 0;
  FERRY_CHECK_ARG(rows == 1 || (stride >= cols && ldc >= blocks * 16 && lds >= blocks),
                  "a row stride is smaller than the row");
  FERRY_CHECK_ARG(ldc % 4 == 0, "the codes' row stride must be a multiple of 4");
  return 0;
}

// rows that follow each other without a gap are one row
void flatten(int64_t* rows, int64_t* cols, int64_t stride, int64_t ldc, int64_t lds) {
  if (*cols % 32 == 0 && stride == *cols && ldc == *cols / 2 && lds == *cols / 32 &&
      *rows * *cols < ((int64_t)1 << 33)) {
    *cols *= *rows;
    *rows = 1;
  }
}

}  // namespace
}  // namespace ferry

using namespace ferry;

extern "C" int ferry_mxfp4_quantize(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t x_stride,
                                    void* codes, int64_t codes_stride, void* scales, int64_t scales_stride,
                                    void* stream) {
  clear_error();
  bool empty = false;
  if (const int rc = check_rows(rows, cols, x_stride, codes_stride, scales_stride, dtype, &empty)) return rc;
  if (empty) return 0;
  FERRY_CHECK_ARG(x && codes && scales, "null pointer argument");
  FERRY_CHECK_ARG((uintptr_t)x % (dtype == FERRY_F32 ? 4 : 2) == 0 && (uintptr_t)codes % 4 == 0,
                  "x must be aligned to its elements, codes to 4 bytes");
  flatten(&rows, &cols, x_stride, codes_stride, scales_stride);
  const int64_t per = ceil_div(cols, 32) * 4, total = rows * per, groups = ceil_div(total, kThreads);
  const dim3 grid((unsigned)(groups < kMaxGrid ? groups : kMaxGrid)), block(kThreads);
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel, auto* p) {
    launch("mxfp4_quantize", kernel, grid, block, 0, s, p, x_stride, cols, (uint32_t)per, total,
           (uint8_t*)codes, codes_stride, (uint8_t*)scales, scales_stride);
  };
  if (dtype == FERRY_BF16) go(mxfp4_quantize_kernel<bf16_t>, (const bf16_t*)x);
  else if (dtype == FERRY_F16) go(mxfp4_quantize_kernel<_Float16>, (const _Float16*)x);
  else go(mxfp4_quantize_kernel<float>, (const float*)x);
  FERRY_LAUNCHED("mxfp4_quantize");
  return 0;
}

extern "C" int ferry_mxfp4_dequantize(const void* codes, int64_t codes_stride, const void* scales,
                                      int64_t scales_stride, int64_t rows, int64_t cols, void* out,
                                      int32_t dtype, int64_t out_stride, void* stream) {
  clear_error();
  bool empty = false;
  if (const int rc = check_rows(rows, cols, out_stride, codes_stride, scales_stride, dtype, &empty)) return rc;
  if (empty) return 0;
  FERRY_CHECK_ARG(out && codes && scales, "null pointer argument");
  FERRY_CHECK_ARG((uintptr_t)out % (dtype == FERRY_F32 ? 4 : 2) == 0 && (uintptr_t)codes % 4 == 0,
                  "out must be aligned to its elements, codes to 4 bytes");
  flatten(&rows, &cols, out_stride, codes_stride, scales_stride);
  const int64_t per = ceil_div(cols, 32) * 4, total = rows * per, groups = ceil_div(total, kThreads);
  const dim3 grid((unsigned)(groups < kMaxGrid ? groups : kMaxGrid)), block(kThreads);
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel, auto* p) {
    launch("mxfp4_dequantize", kernel, grid, block, 0, s, (const uint8_t*)codes, codes_stride,
           (const uint8_t*)scales, scales_stride, cols, (uint32_t)per, total, p, out_stride);
  };
  if (dtype == FERRY_BF16) go(mxfp4_dequantize_kernel<bf16_t>, (bf16_t*)out);
  else if (dtype == FERRY_F16) go(mxfp4_dequantize_kernel<_Float16>, (_Float16*)out);
  else go(mxfp4_dequantize_kernel<float>, (float*)out);
  FERRY_LAUNCHED("mxfp4_dequantize");
  return 0;
}
