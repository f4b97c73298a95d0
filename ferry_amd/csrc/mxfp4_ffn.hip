// Grouped SwiGLU expert FFN over MXFP4 cache slots.
//
// For each expert e with rows p in [starts[e], starts[e+1]):
//   x = in[rows[p]];  g = x Wg^T;  u = x Wu^T;  a = silu(g) * u;  y = a Wd^T;
//   out = bf16(y * w[rows[p], cols[p]])
// with cache[slot] = [codes of Wg (I x H) | Wu (I x H) | Wd (H x I), then their scales], the MXFP4 form
// of the bf16 cache row (mxfp4.hip).  Sums are fp32.  Two kinds of activations:
//  * bf16 (Q = false): x is bf16 and a is rounded to bf16, an operand of the bf16 matrix instruction (in
//    calls of few pairs to 11 bits: small_rows).  The 4-bit weights become bf16 in registers, which is exact.
//  * MXFP4 (Q = true): x is codes and scales, and a is quantised from fp32 in the up epilogue, per 32
//    columns, as mxfp4_quantize does; both products run on the scaled 4-bit matrix instruction.
//
// A lane's 16 bytes of weight codes are one block of 32 along K with one scale.  In a chunk of 128 along K, the lanes
// of row r take the blocks lane / 16 = 0..3: for the 4-bit instruction that is its operand layout, and for
// the bf16 one the four steps s of a chunk multiply the elements 8 s .. 8 s + 7 of the blocks; the order along K
// inside a product is free as long as both operands share it.  So the plain row-major rows are operands
// without any repacking.
//
// Measured, all experts (2048 x 768, 128 of them, top 8, Zipf 1.1): one token 7.0 + 5.6 us (up + down; launch
// latency), 16 tokens 14.6 + 8.2 us, with weights that no cache holds 16.8 + 10.2 (3.2 and 2.7 TB/s of weights), with 4-bit
// activations 12.5 + 7.3 and 15.2 + 8.8; 8,192 tokens 346 + 237 us (1,190 and 870 TFLOP/s, without the 47 experts of at
// most 16 rows 1,240 and 900; a library product of bf16 matrices of 32768 x 2048 x 1536 runs at 1,372), with 4-bit
// activations 178 + 136 (2,300 and 1,510 TFLOP/s).
#include "ffn_common.h"
#include "mxfp4_plan.h"

#include <algorithm>
#include <bitset>
#include <type_traits>

namespace ferry {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kSmallRows = 16;   // experts with at most this many rows run small_rows

struct MxArgs {
  const uint8_t* cache;
  const uint8_t* x;         // bf16 [R, H], or codes [R, H / 2]
  const uint8_t* x_scales;  // [R, H / 32] (Q)
  const bf16_t* w;          // [R, k] routing weights in sorted-ID order
  const int64_t* starts;    // [E+1]
  const int64_t* rows;      // [R*k]
  const int64_t* cols;      // [R*k]
  uint8_t* act;             // bf16 [R*k, I], or codes [R*k, I / 2]
  uint8_t* act_scales;      // [R*k, I / 32] (Q)
  bf16_t* out;              // [R*k, H]
  int64_t H, I, k;
  int32_t out_mode;
  int32_t tile_rows;        // of the tiled kernels: at most theirs
  int32_t known;            // the listed experts' row counts were given
  int32_t fine;             // small_rows
};
struct SmallArgs : MxArgs {
  int32_t items, bufs;      // small_rows
  ExpertList list;
};
struct TiledArgs : MxArgs {
  int32_t tile_wgs;         // workgroups that take tiles; the others take the small experts
  int32_t items;            // small_rows
  ExpertList list, small;
};

// 8 elements of a code word as bf16, scaled (exact)
__device__ __forceinline__ bf16x8 decode8(uint32_t c, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2);
  const bf16x2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3);
  return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}
// the scale of a byte for the conversions, which read the exponent field (0: 2^-127, 255: NaN)
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ floatx4 mma_fp4(u32x4 w, int sw, u32x4 x, int sx, floatx4 c) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 0, sw, 0, sx);
}

typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) const u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) const uint32_t lds_u32;
template <typename T>
__device__ __forceinline__ auto lds_get(uint32_t at) { return *reinterpret_cast<T*>((uintptr_t)at); }

// The weight matrix of a projection in a cache row: codes and scales of `row`, K columns.
struct Weights {
  const uint8_t* codes;
  const uint8_t* scales;
};
// MODE 0: gate (part 0) and up (part 1), rows of H; MODE 1: down, rows of I
template <int MODE>
__device__ __forceinline__ Weights weights_at(const MxArgs& a, int slot, int part, int64_t row) {
  const int64_t n = a.H * a.I;   // elements of a matrix
  const int64_t at = MODE == 0 ? part * n + row * a.H : 2 * n + row * a.I;
  const uint8_t* base = a.cache + (int64_t)slot * (3 * n / 32 * 17);
  return {base + at / 2, base + 3 * n / 2 + at / 32};
}

// a = silu(g) * u quantised: this lane's values v of a block that it shares with the lanes ^ 16, ^ 32
// (each lane 8 of 32 columns); returns the scale byte
__device__ __forceinline__ int block_scale(const float (&v)[8]) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16, 64));
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32, 64));
  const int ex = (int)(amax >> 23);
  return ex == 255 ? 255 : (ex > 2 ? ex - 2 : 0);
}
__device__ __forceinline__ uint32_t block_codes(const float (&v)[8], int byte) {
  const bool bad = byte == 255;
  const float inv = __uint_as_float((uint32_t)(bad ? 0 : 254 - byte) << 23);   // 2^(127 - byte), exact
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = bad ? 0.0f : v[i] * inv;
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, y[0], y[1], 1.0f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2], y[3], 1.0f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[4], y[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[6], y[7], 1.0f, 3);
}

// =============================================================================================
// Experts with at most 16 rows (decode, and the smallest experts of a prefill)
// =============================================================================================

// One workgroup: `items` times 16 NF weight rows (MODE 0: 8 NF columns of gate and of up; MODE 1: 16 NF hidden rows) x
// the expert's rows.  Its four wavefronts split K in units of 256, whose sums meet in LDS in wavefront order.
// Bound by the weight bytes: a wavefront brings its weights by direct loads of whole cache lines (8 rows x
// 128 bytes) into LDS, from where it reads the operands (swizzled as in the tiles below), two units in two
// buffers, from item to item; straight to registers in operand order, the lanes' 64 places of 16 bytes a load
// bound the kernel at 3 TB/s.  The rows' activations go to registers, once for all items where two units hold them:
// only the lanes of rows that are there load.
// 31 experts of 2048 x 768 (16 tokens, Zipf 1.1): up 14.6 us, down 8.2 us (3.5 and 3.2 TB/s, in part from the last-level
// cache), with 4-bit activations 12.5 and 7.3 (4.1 and 3.6; a large copy's rate is 5.2).  The decoding of the weights to
// bf16 is what the 4-bit form saves.
//
// In calls of at most kFinePairs (token, expert) pairs the activations of experts with at most kFineRows rows are not
// rounded to bf16 between up and down: in their 16 bits stand fp16 numbers below 2, and eight columns share the largest
// one's 8-bit exponent, a bit of it in each one's highest exponent bit, which is 0.  A column of down to 2^-14 of the
// largest so has 11 bits and one of down to 2^-17 at least bf16's 8, whatever its neighbours hold; smaller ones are off by at
// most 2^-25 of the largest.  An infinity stays one, a NaN makes eight of them.  Down multiplies the upper 8 bits in the
// rows 0 to 7 of the instruction and the lower three, both exact in bf16, in the rows 8 to 15 that such experts leave
// empty, and adds the two.  An output's mean error is 0.0017 of its size so, its own rounding to bf16, otherwise 0.0023.
// Down of one token takes 5.7 us so, otherwise 4.9; of 8 tokens 8.9 and 7.0; larger calls would pay more for less (16 tokens
// 10.2 us instead of 8.2, error 0.0020: experts of more rows keep bf16).
constexpr int kFineRows = 8, kFinePairs = 64;
constexpr int kUnits = 2;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// The shared exponent e is that of the largest column rounded to 11 bits (255: infinite); e - 1 is stored, with a NaN 255 and
// nothing but ones: its bit 3 - i in column 2 i, its bit 7 - i in column 2 i + 1.
// This lane's four of eight columns, the others in the lane ^ 16: `upper` the last four.
__device__ __forceinline__ u32x2 fine_pack(const float (&v)[4], bool upper) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16, 64));
  const uint32_t e = max((amax + 0x1000u) >> 23, 1u);
  u32x2 y;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const f16x2 n = {(_Float16)__builtin_amdgcn_ldexpf(v[2 * j], 127 - (int)e),
                     (_Float16)__builtin_amdgcn_ldexpf(v[2 * j + 1], 127 - (int)e)};
    const uint32_t k = (e - 1) >> (3 - (j + (upper ? 2 : 0)));
    // an infinity's exponent bits 31 become 15: 2^128
    y[j] = amax > 0x7f800000u ? ~0u : (__builtin_bit_cast(uint32_t, n) & 0xbfffbfffu) | (k & 1u) << 14 | (k >> 4 & 1u) << 30;
  }
  return y;
}
// the eight as bf16: their upper 8 bits, or with `low` the lower three
__device__ __forceinline__ u32x4 fine_unpack(u32x4 c, bool low) {
  uint32_t t = c[0] & 0x40004000u;
#pragma unroll
  for (int i = 1; i < 4; ++i) t |= c[i] >> i & (0x40004000u >> i);
  const uint32_t e = (t >> 11 & 15u) | (t >> 23 & 0xf0u);   // less 1
  const uint32_t bits = (e == 255 ? 0xffffffffu : 0xbfffbfffu) & (low ? ~0u : 0xfff8fff8u);
  const uint32_t upper = low ? bits & 0xfff8fff8u : 0u;
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 part = __builtin_bit_cast(f16x2, c[i] & bits) - __builtin_bit_cast(f16x2, c[i] & upper);
    const uint32_t x0 = __float_as_uint(__builtin_amdgcn_ldexpf((float)part[0], (int)e - 126));
    const uint32_t x1 = __float_as_uint(__builtin_amdgcn_ldexpf((float)part[1], (int)e - 126));
    y[i] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
  }
  return y;
}
__device__ __forceinline__ int swz_w16(int row) { return (row >> 1) & 7; }   // 16 consecutive rows

template <int NF>
constexpr int kUnitBytes = 16 * NF * 136;   // LDS of a unit: codes, scales
template <int NF>
constexpr int kSmallBytes = 4 * kUnits * kUnitBytes<NF>;   // LDS of a workgroup, at most
// bx: number of its first item; bufs: buffers of a wavefront, 1 only for one item of up to one unit a wavefront; tid:
// 0 to 255
template <int MODE, bool Q, int NF>
__device__ __forceinline__ void small_rows(const MxArgs& a, int e, int slot, int bx, int items, int bufs, char* smem,
                                           int tid) {
  constexpr int kRowsW = 16 * NF, kW = kRowsW * 128, kUnit = kUnitBytes<NF>;
  constexpr int kRowsItem = MODE == 0 ? 8 * NF : 16 * NF, kLoads = 2 * NF + NF / 2;   // direct loads of a unit
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int64_t K = MODE == 0 ? a.H : a.I;
  const int chunks = (int)(K / 128), units = (chunks + 1) / 2;
  auto first_unit = [&](int w) { return w * units / 4; };
  const int u0 = first_unit(wave), mine = first_unit(wave + 1) - u0, steps = mine * items;
  const uint32_t lds0 = lds_addr(smem) + (uint32_t)(wave * bufs * kUnit);

  // the loads run over the items' units: the next one's item and unit
  const Weights w0 = weights_at<MODE>(a, slot, 0, (int64_t)bx * kRowsItem);
  int issued = 0, item = 0, unit = 0;
  auto load_next = [&]() {
    if (issued == steps) return;
    const uint32_t dst = lds0 + (uint32_t)((issued & 1) * kUnit);
    const int u = u0 + unit;
    const bool tail = 2 * u + 1 >= chunks;   // half a unit: its other half is read again, not multiplied
    const int64_t row = (int64_t)item * kRowsItem;
    const uint8_t* const codes = w0.codes + row * (K / 2) + u * 128;
#pragma unroll
    for (int j = 0; j < 2 * NF; ++j) {
      const int t = 8 * j + (lane >> 3), part = MODE == 0 ? j / NF : 0;
      const int piece = (lane & 7) ^ swz_w16(t);
      const uint32_t off = (uint32_t)(t - part * 8 * NF) * (uint32_t)(K / 2) + (uint32_t)((tail ? piece & 3 : piece) * 16);
      dma16(reinterpret_cast<const char*>(uniform_ptr(codes + (part ? a.H * a.I / 2 : 0))), off, dst + (uint32_t)(j * 1024));
    }
    const uint8_t* const scales = w0.scales + row * (K / 32) + u * 8;   // 8 bytes a row, two lanes
#pragma unroll
    for (int j = 0; j < NF / 2; ++j) {
      const int t = 32 * j + (lane >> 1), part = MODE == 0 && t >= 8 * NF;
      const uint32_t off = (uint32_t)(t - part * 8 * NF) * (uint32_t)(K / 32) + (tail ? 0u : (uint32_t)((lane & 1) * 4)) +
                           (part ? (uint32_t)(a.H * a.I / 32) : 0u);
      dma4(reinterpret_cast<const char*>(uniform_ptr(scales)), off, dst + (uint32_t)(kW + j * 256));
    }
    ++issued;
    if (++unit == mine) unit = 0, ++item;
  };
  // the first units' weights do not depend on the expert's rows: where those are known to be 1 to 16, their
  // loads go first
  if (a.known)
#pragma unroll 1
    for (int i = 0; i < kUnits; ++i) load_next();
  const int64_t start = a.starts[e];
  const int64_t n = a.starts[e + 1] - start;
  if (n < 1 || n > kSmallRows) {
    wait_cnt<0>();
    return;
  }
  const bool fine = !Q && a.fine && n <= kFineRows;
  const int row = MODE == 1 && fine ? r & 7 : r;
  const bool live = row < n;
  const int64_t p = start + (live ? row : 0);
  const int64_t src = MODE == 0 ? a.rows[p] : p;
  const uint8_t* xp = MODE == 0 ? a.x : a.act;
  const uint8_t* xs = MODE == 0 ? a.x_scales : a.act_scales;
  xp += Q ? src * (K / 2) + q * 16 : src * K * 2 + q * 64;
  if (Q) xs += src * (K / 32) + q;
  constexpr int XL = Q ? 1 : 4;   // 16-byte loads of a lane and chunk
  u32x4 xv[kUnits][2][XL] = {};
  uint32_t xb[kUnits][2] = {};
  auto load_x = [&](int lu) {     // of the units lu, lu + 1 of the wavefront's
    if (live)
#pragma unroll
      for (int b = 0; b < kUnits; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int c = 2 * (u0 + lu + b) + j;
          if (lu + b < mine && c < chunks) {
#pragma unroll
            for (int s = 0; s < XL; ++s) xv[b][j][s] = *(const u32x4*)(xp + (int64_t)c * (Q ? 64 : 256) + s * 16);
            if (Q) xb[b][j] = xs[c * 4];
          }
        }
  };
  int64_t o = 0;
  float wt = 0;
  if constexpr (MODE == 1) {
    const int64_t t = a.rows[p] * a.k + a.cols[p];
    wt = bf16_to_f32(a.w[t]);
    o = a.out_mode == 0 ? t : p;
  }
  load_x(0);
  if (!a.known)
#pragma unroll 1
    for (int i = 0; i < kUnits; ++i) load_next();
  // what was loaded to registers is awaited here: later waits leave the direct loads that they do not need
#pragma unroll
  for (int b = 0; b < kUnits; ++b)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int s = 0; s < XL; ++s) asm volatile("" : "+v"(xv[b][j][s]));
      if (Q) asm volatile("" : "+v"(xb[b][j]));
    }
  if constexpr (MODE == 1) asm volatile("" : "+v"(wt), "+v"(o));
  auto unpack_x = [&]() {
    if constexpr (MODE == 1 && !Q)
      if (fine)
#pragma unroll
        for (int b = 0; b < kUnits; ++b)
          if (b < mine)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int s = 0; s < XL; ++s) xv[b][j][s] = fine_unpack(xv[b][j][s], r >= 8);
  };
  unpack_x();

  int step = 0;
  for (int m = 0; m < items; ++m) {
    floatx4 acc[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[f] = floatx4{0, 0, 0, 0};
    for (int lu = 0; lu < mine; lu += kUnits) {
      if (mine > kUnits && lu + m > 0) load_x(lu), unpack_x();
#pragma unroll
      for (int b = 0; b < kUnits; ++b) {
        if (lu + b >= mine) break;
        if (step > 0) {   // into the last unit's buffer, whose operands or sums have been read
          wait_cnt<63>();
          load_next();
        }
        if (issued > step + 1) wait_cnt<kLoads>();   // the wavefront's own LDS: no barrier
        else wait_cnt<0>();
        const uint32_t at = lds0 + (uint32_t)((step & 1) * kUnit);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (2 * (u0 + lu + b) + j >= chunks) break;
#pragma unroll
          for (int f = 0; f < NF; ++f) {
            const u32x4 c = lds_get<lds_u32x4>(at + (uint32_t)(f * 2048 + r * 128 + (((4 * j + q) ^ swz_w16(r)) << 4)));
            const uint32_t sw = lds_get<lds_u32>(at + (uint32_t)(kW + (f * 16 + r) * 8 + j * 4));
            if constexpr (Q) {
              acc[f] = mma_fp4(c, (int)(sw >> (8 * q)), xv[b][j][0], (int)xb[b][j], acc[f]);
            } else {
              const float sc = scale_of(__builtin_amdgcn_ubfe(sw, 8 * q, 8));
#pragma unroll
              for (int s = 0; s < 4; ++s)
                acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(decode8(c[s], sc), __builtin_bit_cast(bf16x8, xv[b][j][s]),
                                                                 acc[f], 0, 0, 0);
            }
          }
        }
        ++step;
      }
    }
    // a wavefront's sums go where its last unit of the item was
    auto sums_of = [&](int w) {
      const int of = first_unit(w + 1) - first_unit(w), last = of ? (of * (m + 1) - 1) & 1 : 0;
      return lds_addr(smem) + (uint32_t)((w * bufs + last) * kUnit);
    };
    wait_cnt<63>();
#pragma unroll
    for (int f = 0; f < NF; ++f)
      *reinterpret_cast<__attribute__((address_space(3))) floatx4*>((uintptr_t)(sums_of(wave) + (uint32_t)((f * 64 + lane) * 16))) =
          acc[f];
    wait_cnt<63>();
    wg_barrier();
    // lane l of a tile holds the columns (l / 16) * 4 + i of row l % 16
    auto sum = [&](int f) {
      floatx4 v = {};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const floatx4 part = lds_get<__attribute__((address_space(3))) floatx4>(sums_of(w) + (uint32_t)((f * 64 + lane) * 16));
        v = w ? v + part : part;
      }
      return v;
    };
    const int at = bx + m;
    auto next = [&]() {   // the sums are read: their place is free
      if (m + 1 < items) {
        wait_cnt<63>();
        wg_barrier();
      }
    };
    if constexpr (MODE == 0 && Q) {
      static_assert(NF == 4);   // a block of 32 columns
      floatx4 g[2], u[2];       // columns 16 b + 4 q + i
#pragma unroll
      for (int b = 0; b < 2; ++b)
        if (wave == 0) g[b] = sum(b), u[b] = sum(2 + b);
      next();
      if (wave == 0) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = silu_mul(g[i / 4][i & 3], u[i / 4][i & 3]);
        const int byte = block_scale(v);
        const uint32_t c = block_codes(v, byte);
        if (live) {
          uint8_t* o = a.act + p * (a.I / 2) + at * 16 + q * 2;
          *(uint16_t*)o = (uint16_t)c;
          *(uint16_t*)(o + 8) = (uint16_t)(c >> 16);
          if (q == 0) a.act_scales[p * (a.I / 32) + at] = (uint8_t)byte;
        }
      }
    } else if constexpr (MODE == 0) {
      floatx4 g = {}, u = {};
      if (wave < NF / 2) g = sum(wave), u = sum(NF / 2 + wave);
      next();
      if (wave < NF / 2) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = silu_mul(g[i], u[i]);
        const u32x2 y = fine ? fine_pack(v, q & 1) : u32x2{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])};
        if (live) *(u32x2*)(a.act + (p * a.I + at * (8 * NF) + wave * 16 + q * 4) * 2) = y;
      }
    } else {
      static_assert(NF == 4);   // a tile for each wavefront
      floatx4 y = sum(wave);
      next();
      if (fine)   // the lower bits' rows
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] += __shfl_xor(y[i], 8, 64);
      if (live && (!fine || r < 8))
        *(u32x2*)(a.out + o * a.H + at * (16 * NF) + wave * 16 + q * 4) =
            u32x2{pk_bf16(y[0] * wt, y[1] * wt), pk_bf16(y[2] * wt, y[3] * wt)};
    }
  }
}

// weight rows of a workgroup, in tiles of 16
template <int MODE, bool Q>
constexpr int kSmallNF = MODE == 0 && !Q ? 2 : 4;
template <int MODE, bool Q>
__device__ __host__ __forceinline__ int small_cols(const MxArgs& a) {   // items of an expert
  return (int)(MODE == 0 ? a.I / (8 * kSmallNF<0, Q>) : a.H / (16 * kSmallNF<1, Q>));
}

// Down with bf16 activations: within the registers of four workgroups a CU (16 tokens 8.6 us, with three 9.7).
template <int MODE, bool Q>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(MODE == 1 && !Q ? 4 : 1))) void mx_small(SmallArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  small_rows<MODE, Q, kSmallNF<MODE, Q>>(a, a.list.expert[blockIdx.y], a.list.slot[blockIdx.y], blockIdx.x * a.items,
                                         a.items, a.bufs, smem, threadIdx.x);
}

template <int MODE, bool Q>
int small_launch(SmallArgs& a, int64_t cus, hipStream_t s) {
  constexpr int NF = kSmallNF<MODE, Q>;
  const int64_t K = MODE == 0 ? a.H : a.I;
  const int cols = small_cols<MODE, Q>(a);
  // up to one unit a wavefront: one buffer, twice as many workgroups at once (down at 16 tokens, 4-bit activations,
  // 7.0 us, with two items and two buffers 8.2)
  a.items = K > 1024 ? small_items(a.list.n, cols, NF == 2 ? 4 : 2, cus) : 1;
  a.bufs = K > 1024 ? kUnits : 1;
  const dim3 g((unsigned)(cols / a.items), (unsigned)a.list.n);
  launch(MODE == 0 ? "mx_small_up" : "mx_small_down", mx_small<MODE, Q>, g, dim3(256),
         (uint32_t)(kSmallBytes<NF> / kUnits * a.bufs), s, a);
  FERRY_LAUNCHED("mx_small");
  return 0;
}

// =============================================================================================
// Larger experts: tiles of TM rows x TN weight rows
// =============================================================================================

// A wavefront multiplies 8 x 4 tiles of 16 rows x 16 weight rows.  Activations and weights are staged in LDS by
// direct loads.  Loading the weights to registers in operand order instead takes no LDS, but its lanes touch 64
// places of 16 bytes: address processing then bounds the kernels (5 us for 128 along K, whatever the products).
// A row's 16-byte pieces are stored at slot piece ^ swizzle(row), so that the 16 rows that a quarter of a
// wavefront reads lie on 16 different 16-byte bank groups (any LDS read of up to 16 bytes a lane takes the
// same 7 clocks).
//
// The loads run on from tile to tile; the next tile's rows are looked up meanwhile.
// Rows of a tile that hold no row of the expert are not loaded, in steps of a quarter, nor multiplied, from
// half a tile on.
//
// MODE 0: of a wavefront's four weight tiles, two are gate rows and two the up rows of the same 32 columns.
// The weight rows of the two tiles c of 32 columns interleave in groups of four, 8 g + 4 c + [0, 4):
// a lane then holds 8 consecutive output columns of one row.
constexpr int kTileCols = 256;   // weight rows of a large tile: 128 or 256 output columns
template <int MODE, int TN = kTileCols>
constexpr int kOutCols = MODE == 0 ? TN / 2 : TN;
// first weight row (of the tile's) of a wavefront's weight tile f
template <int MODE, int TN = kTileCols>
__device__ __forceinline__ constexpr int wtile(int f) {
  return (f >> 1) * (MODE == 0 ? TN / 2 : 32) + (f & 1) * 4;
}

struct MxTile {
  int64_t row0;        // grouped row of the tile's first row
  int vrows, nt, slot; // its rows (> 0), number of its columns' tile, cache slot
};
__device__ __forceinline__ MxTile mx_locate(const TiledArgs& a, const TileTable& tt, int tile, int ntn) {
  MxTile t;
  const int mt = tile / ntn;
  t.nt = tile - mt * ntn;
  const int li = __builtin_amdgcn_readfirstlane(find_entry(tt, mt));
  const int m0 = (mt - __builtin_amdgcn_readfirstlane(tt.cum[li])) * a.tile_rows;
  t.row0 = uniform64(tt.start[li]) + m0;
  t.vrows = min(__builtin_amdgcn_readfirstlane(tt.rows[li]) - m0, a.tile_rows);
  t.slot = a.list.slot[li];
  return t;
}

// Per tile row, two sets taken in turn: the token, and for MODE 1 the slot index, the output row and the
// routing weight (bf16 bits).
template <int MODE, int TM>
struct __attribute__((aligned(256))) RowTables {
  int32_t row[2][TM], col[MODE == 1 ? 2 : 1][MODE == 1 ? TM : 64], orow[MODE == 1 ? 2 : 1][MODE == 1 ? TM : 64],
      wt[MODE == 1 ? 2 : 1][MODE == 1 ? TM : 64];
  // the tile rows' indices (low words; rows past the last: the first row's) into set p
  __device__ __forceinline__ void load(const MxArgs& a, const MxTile& t, int p, int wave, int lane) {
    if (wave < TM / 64) {
      const int v = 64 * wave + lane;
      const uint32_t off = (uint32_t)((v < t.vrows ? v : 0) * 8);
      dma4(reinterpret_cast<const char*>(uniform_ptr(a.rows + t.row0)), off, lds_addr(row[p]) + 256 * wave);
      if constexpr (MODE == 1)
        dma4(reinterpret_cast<const char*>(uniform_ptr(a.cols + t.row0)), off, lds_addr(col[p]) + 256 * wave);
    }
  }
  // output row and routing weight of the rows of set p, before the epilogue reads them
  __device__ __forceinline__ void outputs(const MxArgs& a, const MxTile& t, int p, int wave, int lane) {
    if (MODE == 1 && wave < TM / 64) {
      const int v = 64 * wave + lane;
      const int64_t tj = (int64_t)row[p][v] * a.k + col[p][v];
      dma2(reinterpret_cast<const char*>(a.w), (uint32_t)(tj * 2), lds_addr(wt[p]) + 256 * wave);
      orow[p][v] = a.out_mode == 0 ? (int32_t)tj : (int32_t)(t.row0 + (v < t.vrows ? v : 0));
    }
  }
};

// a lane's number where what follows from it is to be computed on the spot, not kept through the loops
__device__ __forceinline__ int fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// The sums of a wavefront's tiles into the activations or the outputs: tile i of group wm of WM holds the tile's
// rows 16 (WM i + wm) ..
template <int MODE, bool Q, int WM, int TM, int TN, int MI>
__device__ __forceinline__ void mx_epilogue(const MxArgs& a, const MxTile& t, const RowTables<MODE, TM>& tab, int set,
                                            const floatx4 (&acc)[MI][4], int wm, int wn, int lane_) {
  const int lane = fresh(lane_), r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int row = 16 * (WM * i + wm) + r;
    const bool live = row < t.vrows;
    if constexpr (MODE == 0) {
      float v[8];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * c + j] = silu_mul(acc[i][c][j], acc[i][2 + c][j]);
      const int64_t col = t.nt * kOutCols<0, TN> + wn * 32;
      if constexpr (Q) {
        const int byte = block_scale(v);
        const uint32_t c = block_codes(v, byte);
        if (live) {
          *(uint32_t*)(a.act + (t.row0 + row) * (a.I / 2) + col / 2 + q * 4) = c;
          if (q == 0) a.act_scales[(t.row0 + row) * (a.I / 32) + col / 32] = (uint8_t)byte;
        }
      } else if (live) {
        *(u32x4*)(a.act + ((t.row0 + row) * a.I + col + q * 8) * 2) =
            u32x4{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7])};
      }
    } else if (live) {
      const float wt = __uint_as_float((uint32_t)tab.wt[set][row] << 16);
      bf16_t* const o = a.out + (int64_t)tab.orow[set][row] * a.H + t.nt * kOutCols<1, TN> + wn * 64 + q * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 y;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < 4; j += 2)
            y[2 * c + j / 2] = pk_bf16(acc[i][2 * h + c][j] * wt, acc[i][2 * h + c][j + 1] * wt);
        *(u32x4*)(o + 32 * h) = y;
      }
    }
  }
}

// A workgroup's tile of a round, `total` if it has none.  Workgroup b runs on XCD b % 8, whose workgroups take a run of
// tiles: tiles of one expert follow each other, columns fastest, and share their rows and weights in that XCD's
// L2.  What is left for a last round is spread over the XCDs, so that no CU has two tiles of it where another
// has none (777 tokens, top 6 of 64 experts of 2048 x 1408, up: 72 us; with the rest on the first XCDs 89).
__device__ __forceinline__ int tile_of(int round, int total, int wgs) {
  const int g = wgs, x = (int)(blockIdx.x % 8), j = (int)(blockIdx.x / 8);   // g: a multiple of 8
  const int left = total - round * g;
  if (left >= g) return round * g + x * (g / 8) + j;
  if (left <= 0) return total;
  const int from = left * x / 8, to = left * (x + 1) / 8;
  return j < to - from ? round * g + from + j : total;
}

// bf16 activations.  Four wavefronts share 128 rows; two such workgroups run on a CU, each in its own time, so
// that one's barriers, epilogues and loads fall into the other's products.  A step is 64 along K: rows of 128
// bytes, two buffers, the loads one step ahead; weights in pieces of 128 along K.  The barrier of a step stands before
// its last products, whose operands are in registers by then: behind it the next step's first operands are read, and
// the loads of the freed buffers issued, between those products.
template <int MODE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void mx_tiled16(TiledArgs a) {
  constexpr int NI = 4, W = 4, TM = 128, MI = 8, TN = kTileCols, COLS = kOutCols<MODE>;
  constexpr int RW = 64;                                 // a weight row's bytes in a buffer
  constexpr int kX = TM * 128, kW = TN * RW, kS = TN * 4;   // bytes of a buffer: rows, weights, scales
  constexpr int LX = 4, LW = 4;                          // direct loads of a wavefront for one
  constexpr int kTileBytes = 2 * (kX + kW + kS), kSmall = kSmallBytes<kSmallNF<MODE, false>>;
  __shared__ TileTable tt;
  __shared__ __attribute__((aligned(1024))) char smem[kTileBytes > kSmall ? kTileBytes : kSmall];
  __shared__ RowTables<MODE, TM> tab;
  if ((int)blockIdx.x >= a.tile_wgs) {
    const int per = small_cols<MODE, false>(a) / a.items, b = (int)blockIdx.x - a.tile_wgs, li = b / per;
    small_rows<MODE, false, kSmallNF<MODE, false>>(a, a.small.expert[li], a.small.slot[li], (b - li * per) * a.items, a.items,
                                                   kUnits, smem, threadIdx.x);
    return;
  }
  build_tile_table<kSmallRows>(a, tt, (uint32_t)a.tile_rows);
  const int64_t K = MODE == 0 ? a.H : a.I;
  const int ntn = (int)((MODE == 0 ? a.I : a.H) / COLS);
  const int total = __builtin_amdgcn_readfirstlane(tt.total) * ntn;
  const int lane = threadIdx.x & 63, wn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int chunks = (int)(K / 128);
  const uint32_t smem0 = lds_addr(smem), wbuf = smem0 + 2 * kX, sbuf = wbuf + 2 * kW;
  const char* const xbase = reinterpret_cast<const char*>(MODE == 0 ? a.x : a.act);
  auto swz_x = [](int row) { return (row >> 1) & 7; };
  auto swz_w = [](int row) { return (row >> 3) & 3; };
  // fragment reads: addresses of tile 0, the others at constant offsets
  const int wrow = (MODE == 0 ? wn * 32 : wn * 64) + 8 * (r >> 2) + (r & 3);
  const uint32_t xa = smem0 + (uint32_t)(r * 128 + (((2 * q) ^ swz_x(r)) << 4));
  const uint32_t wa = wbuf + (uint32_t)(wrow * RW + (((q >> 1) ^ swz_w(wrow)) << 4) + (q & 1) * 8);
  const uint32_t wsa = sbuf + (uint32_t)(wn * 256 + r * 16);
  constexpr int kXTile = 16 * 128;

  // The tile whose steps are being loaded.  Load j of a wavefront moves 1 KiB of rows in a row's order of
  // slots: 8 rows of 128 bytes or 16 of 64.  Load j of the activations moves rows 32 j .. over all wavefronts.
  uint32_t xoff[LX], woff, soff;
  const char *wbase[2], *sbase;   // MODE 0: gate rows (the first half of the loads), up rows
  int xloads = LX;
  auto aim = [&](const MxTile& t, int p) {
    const int l = fresh(lane);
    xloads = min((t.vrows + 31) / 32, LX);
#pragma unroll
    for (int j = 0; j < LX; ++j) {
      const int v = 8 * (W * j + wn) + l / 8;
      const uint32_t src = MODE == 0 ? (uint32_t)tab.row[p][v] : (uint32_t)(t.row0 + (v < t.vrows ? v : 0));
      xoff[j] = (src * (uint32_t)K + (uint32_t)(((l & 7) ^ swz_x(v)) * 8)) * 2u;
    }
    const Weights m0 = weights_at<MODE>(a, t.slot, 0, t.nt * COLS);
    const Weights m1 = weights_at<MODE>(a, t.slot, MODE == 0 ? 1 : 0, MODE == 0 ? t.nt * COLS : t.nt * COLS + TN / 2);
    wbase[0] = reinterpret_cast<const char*>(uniform_ptr(m0.codes));
    wbase[1] = reinterpret_cast<const char*>(uniform_ptr(m1.codes));
    const int v = 16 * wn + l / 4;   // load j: 64 j rows on, in the same order of slots
    woff = (uint32_t)v * (uint32_t)(K / 2) + (uint32_t)(((l & 3) ^ swz_w(v)) * 16);
    // scales: those of a lane's four weight tiles adjacent
    const int row = 8 * (l >> 4) + ((l >> 2) & 3), f = l & 3;
    sbase = reinterpret_cast<const char*>(uniform_ptr(m0.scales));
    soff = (uint32_t)(wn * (MODE == 0 ? 32 : 64) + row + (MODE == 0 ? (f & 1) * 4 : wtile<1>(f))) * (uint32_t)(K / 32) +
           (MODE == 0 && f >= 2 ? (uint32_t)(a.H * a.I / 32) : 0u);
  };
  auto load_x = [&](int j, int n, int b) {   // load j of step n of the loaded tile into buffer b
    if (j < xloads) dma16(xbase + (int64_t)n * 128, xoff[j], smem0 + (uint32_t)(b * kX + (W * j + wn) * 1024));
  };
  auto load_w = [&](int j, int c, int b) {   // of 128 along K number c
    dma16(wbase[j >> 1] + (j & 1) * 32 * K + (int64_t)c * RW, woff, wbuf + (uint32_t)(b * kW + (W * j + wn) * 1024));
  };
  auto load_s = [&](int c, int b) { dma4(sbase + (int64_t)c * 4, soff, sbuf + (uint32_t)(b * kS + wn * 256)); };

  int tile = tile_of(0, total, a.tile_wgs);
  if (tile >= total) return;
  MxTile cur = mx_locate(a, tt, tile, ntn);
  tab.load(a, cur, 0, wn, lane);

  // read ahead: the next step's weights and scales, its first fragments
  u32x2 wr[NI];
  u32x4 wsc, xf[4];
  auto read_x = [&](int to, int s, int i, int b) {   // half s, tile i of the step in buffer b
    xf[to] = lds_get<lds_u32x4>(((xa + (uint32_t)(b * kX)) ^ (uint32_t)(s << 4)) + (uint32_t)(kXTile * i));
  };
  auto read_w = [&](int h, int w) {                  // half h of the 128 along K in buffer w
    const uint32_t at = (wa + (uint32_t)(w * kW)) ^ (uint32_t)(h << 5);
#pragma unroll
    for (int f = 0; f < NI; ++f) wr[f] = lds_get<lds_u32x2>(at + (uint32_t)(wtile<MODE>(f) * RW));
    wsc = lds_get<lds_u32x4>(wsa + (uint32_t)(w * kS));
  };
  int set = 0, wb = 0;   // set of row tables; buffer of the present weights
  bool primed = false;   // the tile's first steps are loaded, its first operands read
  for (int round = 1, later; tile < total; tile = later, ++round, set ^= 1) {
    // the tile after this one; after the last tile its own first steps are loaded again
    later = tile_of(round, total, a.tile_wgs);
    const MxTile next = later < total ? mx_locate(a, tt, later, ntn) : cur;
    const bool few = cur.vrows <= TM / 2;
    if (few || !primed) {
      wait_cnt<0>();   // the tile's row table has landed; the buffers are free behind the barrier
      wg_barrier();
      aim(cur, set);
      wb = 0;
    }
    tab.load(a, next, set ^ 1, wn, lane);
    tab.outputs(a, cur, set, wn, lane);
    if (!few && !primed) {
#pragma unroll
      for (int j = 0; j < LX; ++j) load_x(j, 0, 0), load_x(j, 1, 1);
#pragma unroll
      for (int j = 0; j < LW; ++j) load_w(j, 0, 0);
      load_s(0, 0);
      wait_cnt<0>();
      wg_barrier();
      read_w(0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) read_x(i, 0, i, 0);
    }
    floatx4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int f = 0; f < NI; ++f) acc[i][f] = floatx4{0, 0, 0, 0};
    // one of 32 along K of step h: half a weight tile's 8 elements a lane
    u32x4 wv[2][NI];
    auto decode = [&](int h, int s, int part) {
      const int f = part >> 1, half = part & 1;
      const float sc = scale_of(__builtin_amdgcn_ubfe(wsc[f], 16 * h + 8 * (q >> 1), 8));
      const uint32_t v = wr[f][s];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bf16x2 d = half ? (j ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc, 3)
                                   : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc, 2))
                              : (j ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc, 1)
                                   : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc, 0));
        wv[s][f][2 * half + j] = __builtin_bit_cast(uint32_t, d);
      }
    };
    // Up to 64 rows: a tile of these waits for its loads, not for products.  The rows' buffers hold 128 along K of
    // ROWS tiles, two halves, so that a barrier comes every 128 along K with the loads as far ahead: one
    // tile of up to 32 rows takes 15 us for 2048 along K, with the loop below 22.
    auto loop_few = [&](auto rows) {
      constexpr int ROWS = decltype(rows)::value, XH = ROWS / 2;   // loads of a half
      auto load = [&](int p, int c, int b) {                       // part p of 4 of 128 along K number c
        if (p < 2 * XH)
          dma16(xbase + (int64_t)(2 * c + p / XH) * 128, xoff[p % XH],
                smem0 + (uint32_t)(b * kX + (p / XH) * (kX / 2) + (W * (p % XH) + wn) * 1024));
        load_w(p, c, b);
        if (p == 3) load_s(c, b);
      };
      auto read = [&](int to, int m, int h, int b) {   // fragment m of half h
        xf[to] = lds_get<lds_u32x4>(((xa + (uint32_t)(b * kX + h * (kX / 2))) ^ (uint32_t)((m / ROWS) << 4)) +
                                    (uint32_t)(kXTile * (m % ROWS)));
      };
#pragma unroll
      for (int p = 0; p < 4; ++p) load(p, 0, 0);
      if (chunks > 1)
#pragma unroll
        for (int p = 0; p < 4; ++p) load(p, 1, 1);
      wait_cnt<0>();
      wg_barrier();
      read_w(0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) read(i, i, 0, 0);
      for (int c = 0; c < chunks; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int part = 0; part < 2 * NI; ++part) decode(h, 0, part);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int n = 0; n < 2 * ROWS; ++n) {
            const int s = n / ROWS, i = n % ROWS, k = n - (2 * ROWS - 4);
            if (s == 0)
#pragma unroll
              for (int part = i * 2 * NI / ROWS; part < (i + 1) * 2 * NI / ROWS; ++part) decode(h, 1, part);
            if (n == ROWS) {   // the weights are decoded
              if (h == 1) {
                wait_cnt<0>();   // the next loads have landed, this buffer's fragments are read
                wg_barrier();
                wb ^= 1;
              }
              read_w(h ^ 1, wb);
            }
#pragma unroll
            for (int f = 0; f < NI; ++f)
              acc[i][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[s][f]),
                                                                 __builtin_bit_cast(bf16x8, xf[n & 3]), acc[i][f], 0, 0, 0);
            if (k < 0) read(n & 3, n + 4, h, wb);
            else if (h == 0 || n >= ROWS) read(n & 3, k, h ^ 1, wb);
            if (h == 1 && n >= ROWS) {   // behind the barrier; with two tiles the reads of the first two, too
              if (ROWS == 2) read(n - 2, k - 2, 0, wb);
              if (c + 2 < chunks)
#pragma unroll
                for (int p = (n - ROWS) * 4 / ROWS; p < (n - ROWS + 1) * 4 / ROWS; ++p) load(p, c + 2, wb ^ 1);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    };
    // ROWS: tiles of 16 rows that are multiplied; the others hold no row of the expert
    auto loop = [&](auto rows) {
      constexpr int ROWS = decltype(rows)::value;
      for (int c = 0; c < chunks; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // the first 32 along K are decoded here, the second 32 between the products of the first
#pragma unroll
          for (int part = 0; part < 2 * NI; ++part) decode(h, 0, part);
          __builtin_amdgcn_sched_barrier(0);
          const bool last = c == chunks - 1;
#pragma unroll
          for (int n = 0; n < 2 * ROWS; ++n) {
            const int s = n / ROWS, i = n % ROWS, k = n - (2 * ROWS - 4);
            if (k == 0) {
              wait_cnt<0>();   // the next step's loads have landed, this one's fragments are read
              wg_barrier();
              if (h == 0 && last) aim(next, set ^ 1);
              if (h == 1) wb ^= 1;
              read_w(h ^ 1, wb);
            }
            if (s == 0)
#pragma unroll
              for (int part = i * 2 * NI / ROWS; part < (i + 1) * 2 * NI / ROWS; ++part) decode(h, 1, part);
#pragma unroll
            for (int f = 0; f < NI; ++f)
              acc[i][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[s][f]),
                                                                 __builtin_bit_cast(bf16x8, xf[n & 3]), acc[i][f], 0, 0, 0);
            // the fragment four products on, of this step or the next
            if (k < 0) read_x(n & 3, (n + 4) / ROWS, (n + 4) % ROWS, h);
            else read_x(n & 3, 0, k, h ^ 1);
            if (k >= 0) {   // the loads of the buffers that are free now
              load_x(k, last ? h : 2 * c + 2 + h, h);
              if (h == 0) load_w(k, last ? 0 : c + 1, wb ^ 1);
              if (h == 0 && k == 3) load_s(last ? 0 : c + 1, wb ^ 1);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    };
    if (cur.vrows > TM / 4 * 3) loop(std::integral_constant<int, MI>{});
    else if (cur.vrows > TM / 2) loop(std::integral_constant<int, MI / 4 * 3>{});
    else if (cur.vrows > TM / 4) loop_few(std::integral_constant<int, MI / 2>{});
    else loop_few(std::integral_constant<int, MI / 4>{});
    primed = !few;
    mx_epilogue<MODE, false, 1, TM, TN, MI>(a, cur, tab, set, acc, 0, wn, lane);
    cur = next;
  }
  wait_cnt<0>();   // no load may write this workgroup's LDS after its end
}

// 4-bit activations.  LARGE: eight wavefronts in two rows share 256 x 256, one workgroup on a CU; else four share 128 x
// 128, two workgroups on a CU, each in its own time.  A step is 256 along K: rows of 128 bytes of activations
// and of weights, whole cache lines (with lines of 64 bytes loaded up to three steps ahead, 90 us instead of 70 at
// 32,768 rows x 2048 x 768 up: a CU receives about 64 bytes a clock, in lines of 128), two buffers, the loads
// one step ahead.  Here the barrier stands at a step's end: before its last products, as above, it took 69 to 78 us,
// with scales for two steps at a time 74.  The large tiles load and read half and two thirds as much for
// each product (32,768 rows: 70 us against 86); the small ones' epilogues and waits fall into the other workgroup's products.
template <int MODE, bool LARGE>
__global__ __launch_bounds__(LARGE ? 512 : 256) __attribute__((amdgpu_waves_per_eu(2, 2))) void mx_tiled4(TiledArgs a) {
  constexpr int WM = 2, WN = LARGE ? 4 : 2, MI = LARGE ? 8 : 4, NI = 4, W = WM * WN;
  constexpr int TM = 16 * WM * MI, TN = 64 * WN, COLS = kOutCols<MODE, TN>;
  constexpr int kX = TM * 128, kW = TN * 128;            // bytes of a buffer
  constexpr int LX = 4, LW = 4;                          // direct loads of a wavefront for one
  constexpr int kS = (TN + TM) * 8;                      // scale bytes of a step: weight rows, activation rows
  constexpr int kTileBytes = 2 * (kX + kW + kS), kSmall = W / 4 * kSmallBytes<kSmallNF<MODE, true>>;
  __shared__ TileTable tt;
  __shared__ __attribute__((aligned(1024))) char smem[kTileBytes > kSmall ? kTileBytes : kSmall];
  __shared__ RowTables<MODE, TM> tab;
  if ((int)blockIdx.x >= a.tile_wgs) {
    const int per = small_cols<MODE, true>(a) / (W / 4 * a.items), b = (int)blockIdx.x - a.tile_wgs, li = b / per;
    const int part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);   // LARGE: two workgroups' work of one expert
    small_rows<MODE, true, kSmallNF<MODE, true>>(a, a.small.expert[li], a.small.slot[li],
                                                 (W / 4 * (b - li * per) + part) * a.items, a.items, kUnits,
                                                 smem + part * (kSmall / (W / 4)), threadIdx.x & 255);
    return;
  }
  build_tile_table<kSmallRows>(a, tt, (uint32_t)a.tile_rows);
  const int64_t K = MODE == 0 ? a.H : a.I;
  const int ntn = (int)((MODE == 0 ? a.I : a.H) / COLS);
  const int total = __builtin_amdgcn_readfirstlane(tt.total) * ntn;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int r = lane & 15, q = lane >> 4;
  const int chunks = (int)(K / 128), steps = (chunks + 1) / 2;
  const uint32_t smem0 = lds_addr(smem), wbuf = smem0 + 2 * kX, sbuf = wbuf + 2 * kW;
  const char* const xbase = reinterpret_cast<const char*>(MODE == 0 ? a.x : a.act);
  auto swz_x = [](int row) { return (row >> 1) & 7; };
  auto swz_w = [](int row) { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); };
  // fragment reads: addresses of tile 0, the others at constant offsets
  const int xrow = 16 * wm + r, wrow = (MODE == 0 ? wn * 32 : wn * 64) + 8 * (r >> 2) + (r & 3);
  const uint32_t xa = smem0 + (uint32_t)(xrow * 128 + ((q ^ swz_x(xrow)) << 4));
  const uint32_t wa = wbuf + (uint32_t)(wrow * 128 + ((q ^ swz_w(wrow)) << 4));
  const uint32_t xsa = sbuf + (uint32_t)((TN + xrow) * 8), wsa = sbuf + (uint32_t)(wrow * 8);
  constexpr int kXTile = 16 * WM * 128;

  // The tile whose steps are being loaded.  Load j of a wavefront moves 8 rows of 128 bytes in a row's order of
  // slots; rows 64 j .. over all wavefronts.  A thread moves the scales of one row, a weight or activation row.
  uint32_t xoff[LX], woff;
  const char* wbase[2];   // MODE 0: gate rows (the first half of the loads), up rows
  const uint8_t* sp = nullptr;
  int xloads = LX;
  auto aim = [&](const MxTile& t, int p) {
    const int l = fresh(lane);
    auto src_row = [&](int v) {
      return MODE == 0 ? (uint32_t)tab.row[p][v] : (uint32_t)(t.row0 + (v < t.vrows ? v : 0));
    };
    xloads = min((t.vrows + 8 * W - 1) / (8 * W), LX);
#pragma unroll
    for (int j = 0; j < LX; ++j) {
      const int v = 8 * (W * j + wave) + l / 8;
      xoff[j] = src_row(v) * (uint32_t)(K / 2) + (uint32_t)(((l & 7) ^ swz_x(v)) * 16);
    }
    const Weights m0 = weights_at<MODE>(a, t.slot, 0, t.nt * COLS);
    const Weights m1 = weights_at<MODE>(a, t.slot, MODE == 0 ? 1 : 0, MODE == 0 ? t.nt * COLS : t.nt * COLS + TN / 2);
    wbase[0] = reinterpret_cast<const char*>(uniform_ptr(m0.codes));
    wbase[1] = reinterpret_cast<const char*>(uniform_ptr(m1.codes));
    const int v = 8 * wave + l / 8;   // load j: 64 j rows on, in the same order of slots
    woff = (uint32_t)v * (uint32_t)(K / 2) + (uint32_t)(((l & 7) ^ swz_w(v)) * 16);
    if (wave < W / 2) {
      sp = (wave < W / 4 ? m0.scales : m1.scales) + (int64_t)(64 * (wave & (W / 4 - 1)) + l) * (K / 32);
    } else {
      sp = (MODE == 0 ? a.x_scales : a.act_scales) + (int64_t)src_row(64 * (wave - W / 2) + l) * (K / 32);
    }
  };
  // Where the number of chunks is odd, the last step's rows end in its middle: the lanes of the second half
  // read the first half again (it is not multiplied).
  auto tail = [&](int piece) { return (uint32_t)((piece & 4) << 4); };
  auto load_x = [&](int j, int n, int b) {   // load j of step n of the loaded tile into buffer b
    if (j >= xloads) return;
    uint32_t off = xoff[j];
    if (2 * n + 1 >= chunks) {
      const int l = fresh(lane);
      off -= tail((l & 7) ^ swz_x(8 * (W * j + wave) + l / 8));
    }
    dma16(xbase + (int64_t)n * 128, off, smem0 + (uint32_t)(b * kX + (W * j + wave) * 1024));
  };
  auto load_w = [&](int j, int n, int b) {
    uint32_t off = woff;
    if (2 * n + 1 >= chunks) {
      const int l = fresh(lane);
      off -= tail((l & 7) ^ swz_w(8 * wave + l / 8));
    }
    dma16(wbase[j >> 1] + (j & 1) * (4 * W) * K + (int64_t)n * 128, off, wbuf + (uint32_t)(b * kW + (W * j + wave) * 1024));
  };
  u32x2 sv = {0, 0};
  auto load_s = [&](int n) {
    if (2 * n + 1 < chunks) __builtin_memcpy(&sv, sp + n * 8, 8);
    else __builtin_memcpy(&sv, sp + n * 8, 4);
  };
  auto store_s = [&](int b) {
    *reinterpret_cast<__attribute__((address_space(3))) u32x2*>((uintptr_t)(sbuf + (uint32_t)(b * kS + tid * 8))) = sv;
  };

  int tile = tile_of(0, total, a.tile_wgs);
  if (tile >= total) return;
  MxTile cur = mx_locate(a, tt, tile, ntn);
  tab.load(a, cur, 0, wave, lane);
  wait_cnt<0>();
  wg_barrier();
  aim(cur, 0);
  load_s(0);
#pragma unroll
  for (int j = 0; j < LW; ++j) load_w(j, 0, 0);
#pragma unroll
  for (int j = 0; j < LX; ++j) load_x(j, 0, 0);
  store_s(0);
  wait_cnt<0>();
  wg_barrier();
  int set = 0, b = 0;   // set of row tables; buffer of the present step
  for (int round = 1, later; tile < total; tile = later, ++round, set ^= 1) {
    // the tile after this one; after the last tile its own first step is loaded again
    later = tile_of(round, total, a.tile_wgs);
    const MxTile next = later < total ? mx_locate(a, tt, later, ntn) : cur;
    tab.load(a, next, set ^ 1, wave, lane);
    tab.outputs(a, cur, set, wave, lane);
    floatx4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int f = 0; f < NI; ++f) acc[i][f] = floatx4{0, 0, 0, 0};
    // ROWS: tiles of 16 rows of a wavefront that are multiplied; the others hold no row of the expert
    auto loop = [&](auto rows) {
      constexpr int ROWS = decltype(rows)::value;
      for (int st = 0; st < steps; ++st, b ^= 1) {
        const uint32_t xb = xa + (uint32_t)(b * kX), wb = wa + (uint32_t)(b * kW);
        const uint32_t xsb = xsa + (uint32_t)(b * kS), wsb = wsa + (uint32_t)(b * kS);
        // fragments are read two ahead of their products
        u32x4 xn[2], wf[NI];
        uint32_t xsn[2], wsf[NI];
        auto read_x = [&](int j, int i) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            xn[v] = lds_get<lds_u32x4>((xb ^ (uint32_t)(j << 6)) + (uint32_t)(kXTile * (i + v)));
            xsn[v] = lds_get<lds_u32>(xsb + (uint32_t)(16 * WM * 8 * (i + v) + 4 * j));
          }
        };
        auto read_w = [&](int j) {
#pragma unroll
          for (int f = 0; f < NI; ++f) {
            wf[f] = lds_get<lds_u32x4>((wb ^ (uint32_t)(j << 6)) + (uint32_t)(wtile<MODE, TN>(f) * 128));
            wsf[f] = lds_get<lds_u32>(wsb + (uint32_t)(wtile<MODE, TN>(f) * 8 + 4 * j));
          }
        };
        read_w(0);
        read_x(0, 0);
        const bool last = st + 1 == steps;
        if (last) {   // the loads turn to the next tile
          if (steps == 1) {   // its row indices may still be on their way
            wait_cnt<0>();
            wg_barrier();
          }
          aim(next, set ^ 1);
        }
        const int ls = last ? 0 : st + 1;
        load_s(ls);
#pragma unroll
        for (int j = 0; j < LW; ++j) load_w(j, ls, b ^ 1);
#pragma unroll
        for (int j = 0; j < LX; ++j) load_x(j, ls, b ^ 1);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (j == 1 && 2 * st + 1 >= chunks) break;
          u32x4 cw[NI];
          int cs[NI];
#pragma unroll
          for (int f = 0; f < NI; ++f) cw[f] = wf[f], cs[f] = (int)(wsf[f] >> (8 * q));
#pragma unroll
          for (int i = 0; i < ROWS; i += 2) {
            const u32x4 x0 = xn[0], x1 = xn[1];
            const int s0 = (int)(xsn[0] >> (8 * q)), s1 = (int)(xsn[1] >> (8 * q));
            if (i + 2 < ROWS) {
              read_x(j, i + 2);
            } else if (j == 0) {
              read_x(1, 0);
              read_w(1);
            }
#pragma unroll
            for (int f = 0; f < NI; ++f) acc[i][f] = mma_fp4(cw[f], cs[f], x0, s0, acc[i][f]);
#pragma unroll
            for (int f = 0; f < NI; ++f) acc[i + 1][f] = mma_fp4(cw[f], cs[f], x1, s1, acc[i + 1][f]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        store_s(b ^ 1);
        wait_cnt<0>();   // the next step's loads have landed, this one's fragments are read
        wg_barrier();
      }
    };
    if (LARGE && cur.vrows <= TM / 4) loop(std::integral_constant<int, LARGE ? MI / 4 : MI>{});
    else if (cur.vrows <= TM / 2) loop(std::integral_constant<int, MI / 2>{});
    else if (LARGE && cur.vrows <= TM / 4 * 3) loop(std::integral_constant<int, LARGE ? MI / 4 * 3 : MI>{});
    else loop(std::integral_constant<int, MI>{});
    mx_epilogue<MODE, true, WM, TM, TN, MI>(a, cur, tab, set, acc, wm, wn, lane);
    cur = next;
  }
  wait_cnt<0>();   // no load may write this workgroup's LDS after its end
}

int device_cus(int* cus) {
  int dev = 0;
  FERRY_HIP(hipGetDevice(&dev));
  FERRY_HIP(hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev));
  if (*cus <= 0) *cus = 256;
  return 0;
}

// The launches of a.list and a.small in one kind of activations, as plan_tiles cuts them.  tiles: the row tiles of 256,
// 128 and 64 rows of the experts with more than kSmallRows rows (upper bounds).
template <bool Q>
int launch_lists(TiledArgs& a, const int64_t (&tiles)[3], int32_t phases, int64_t cus, int64_t spare, hipStream_t s) {
  for (int mode = 0; mode < 2; ++mode) {
    if (!(phases & (1 << mode))) continue;
    if (tiles[0]) {
      const int64_t cols = mode == 0 ? a.I / kOutCols<0> : a.H / kOutCols<1>;
      const MxPlan p = plan_tiles(Q, cols, tiles, a.small.n, mode == 0 ? small_cols<0, Q>(a) : small_cols<1, Q>(a), cus, spare);
      a.tile_rows = p.tile_rows;
      a.tile_wgs = p.tile_wgs;
      a.items = p.items;
      const dim3 grid((unsigned)(p.tile_wgs + p.small_wgs)), block(p.large ? 512 : 256);
      const char* const name = mode == 0 ? "mx_tiled_up" : "mx_tiled_down";
      if constexpr (!Q) launch(name, mode == 0 ? mx_tiled16<0> : mx_tiled16<1>, grid, block, 0, s, a);
      else if (p.large) launch(name, mode == 0 ? mx_tiled4<0, true> : mx_tiled4<1, true>, grid, block, 0, s, a);
      else launch(name, mode == 0 ? mx_tiled4<0, false> : mx_tiled4<1, false>, grid, block, 0, s, a);
      FERRY_LAUNCHED("mx_tiled");
      if (p.small_wgs) continue;
    }
    if (a.small.n) {
      SmallArgs b;
      (MxArgs&)b = a;
      b.list = a.small;
      if (const int rc = mode == 0 ? small_launch<0, Q>(b, cus, s) : small_launch<1, Q>(b, cus, s)) return rc;
    }
  }
  return 0;
}

}  // namespace
}  // namespace ferry

using namespace ferry;

extern "C" int ferry_mxfp4_expert_ffn(const void* cache, int64_t cache_rows, int64_t hidden, int64_t inter,
                                      const void* x, const void* x_scales, int64_t rows_in, int64_t topk,
                                      const void* w_sorted, const int64_t* starts, const int64_t* rows,
                                      const int64_t* cols, const int32_t* expert_list, int32_t n_list,
                                      const int32_t* slot_of, int64_t experts, int64_t max_rows_per_expert,
                                      int64_t min_rows_per_expert, const int32_t* list_rows, void* act,
                                      void* out, int32_t out_mode, int32_t phases, int32_t spare_cus,
                                      void* stream) {
  clear_error();
  FERRY_CHECK_ARG(phases >= 1 && phases <= 3, "phases must be 1 (up), 2 (down) or 3 (both)");
  FERRY_CHECK_ARG(hidden > 0 && hidden % 128 == 0, "hidden must be a positive multiple of 128");
  FERRY_CHECK_ARG(inter > 0 && inter % 128 == 0, "intermediate must be a positive multiple of 128");
  FERRY_CHECK_ARG(hidden <= 1 << 20 && inter <= 1 << 20, "hidden and intermediate must be at most 2^20");
  FERRY_CHECK_ARG(topk >= 1 && rows_in >= 0 && n_list >= 0, "bad sizes");
  if (list_rows && max_rows_per_expert == -1) {
    max_rows_per_expert = 0;
    min_rows_per_expert = n_list ? list_rows[0] : 0;
    for (int32_t i = 0; i < n_list; ++i) {
      if (list_rows[i] > max_rows_per_expert) max_rows_per_expert = list_rows[i];
      if (list_rows[i] < min_rows_per_expert) min_rows_per_expert = list_rows[i];
    }
  }
  FERRY_CHECK_ARG(max_rows_per_expert >= 0, "bad sizes");
  FERRY_CHECK_ARG(min_rows_per_expert >= 0 && min_rows_per_expert <= max_rows_per_expert,
                  "min_rows_per_expert must be in [0, max_rows_per_expert]");
  FERRY_CHECK_ARG(experts >= 1 && experts <= FERRY_MAX_EXPERTS, "experts must be in [1, %d]",
                  FERRY_MAX_EXPERTS);
  FERRY_CHECK_ARG(out_mode == 0 || out_mode == 1, "out_mode must be 0 or 1");
  FERRY_CHECK_ARG(spare_cus >= 0 && spare_cus <= 128, "spare_cus must be in [0, 128]");
  FERRY_CHECK_ARG(hidden % 256 == 0 || max_rows_per_expert <= kSmallRows,
                  "hidden must be a multiple of 256 when an expert has more than %d rows", kSmallRows);
  FERRY_CHECK_ARG(rows_in < (int64_t)1 << 31 && topk < (int64_t)1 << 31 && rows_in * topk < (int64_t)1 << 31,
                  "rows*topk must be < 2^31");
  // the kernels address activations with 32-bit byte offsets
  FERRY_CHECK_ARG(rows_in < ((int64_t)1 << 31) / hidden && rows_in * topk < ((int64_t)1 << 31) / inter,
                  "x / act must hold fewer than 2^31 elements");
  // and scales with 32-bit ones from a matrix of the expert's cache row
  FERRY_CHECK_ARG(hidden * inter < ((int64_t)1 << 32), "hidden * intermediate must be under 2^32");
  if (n_list == 0 || rows_in == 0) return 0;
  FERRY_CHECK_ARG(cache && x && w_sorted && starts && rows && cols && expert_list && slot_of && act && out,
                  "null pointer argument");
  FERRY_CHECK_ARG(((uintptr_t)cache | (uintptr_t)x | (uintptr_t)act | (uintptr_t)out) % 16 == 0,
                  "cache, x, act and out must be 16-byte aligned");
  FERRY_CHECK_ARG((uintptr_t)x_scales % 4 == 0, "x_scales must be 4-byte aligned");
  std::bitset<FERRY_MAX_EXPERTS> seen;
  int64_t listed = 0;   // pairs of the listed experts; one may be listed twice
  for (int32_t i = 0; i < n_list; ++i) {
    const int32_t e = expert_list[i];
    FERRY_CHECK_ARG(e >= 0 && e < experts, "expert_list[%d] = %d out of range", i, e);
    const int32_t s = slot_of[e];
    FERRY_CHECK_ARG(s >= 0 && s < cache_rows, "expert %d is not cached (slot %d)", e, s);
    if (list_rows)
      FERRY_CHECK_ARG(list_rows[i] >= min_rows_per_expert && list_rows[i] <= max_rows_per_expert,
                      "list_rows[%d] = %d outside [min_rows_per_expert, max_rows_per_expert]", i,
                      list_rows[i]);
    if (list_rows && !seen[e]) listed += list_rows[i];
    seen[e] = true;
  }
  FERRY_CHECK_ARG(listed <= rows_in * topk, "list_rows name more than rows * topk pairs");
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  const bool quantised = x_scales != nullptr;
  const int64_t pairs = rows_in * topk;
  TiledArgs a;
  a.cache = (const uint8_t*)cache;
  a.x = (const uint8_t*)x;
  a.x_scales = (const uint8_t*)x_scales;
  a.w = (const bf16_t*)w_sorted;
  a.starts = starts;
  a.rows = rows;
  a.cols = cols;
  a.act = (uint8_t*)act;
  a.act_scales = (uint8_t*)act + pairs * (inter / 2);
  a.out = (bf16_t*)out;
  a.H = hidden;
  a.I = inter;
  a.k = topk;
  a.out_mode = out_mode;
  a.known = list_rows != nullptr;
  a.fine = pairs <= kFinePairs;
  // Small experts and the others, each up to kListMax of a launch; without row counts every expert is in both, and the
  // kernels pass over those of the other kind by the device's starts.  An expert's own rows (and with a.fine the call's
  // pairs) decide, so that its results do not depend on which experts are listed with it (the two kinds sum in different
  // orders): with all experts in tiles wherever one has more than kSmallRows rows, 512 tokens (128 experts of 2048 x
  // 768, top 8, Zipf 1.1) took 10 and 5 % less (bf16 and 4-bit activations), 8,192 tokens 1 and 3 %, when the small ones
  // had launches of their own.
  struct Entry {
    int32_t rows, expert;
  } entry[kListMax];
  const bool any[2] = {min_rows_per_expert <= kSmallRows, max_rows_per_expert > kSmallRows};   // small, others
  int32_t at[2] = {any[0] ? 0 : n_list, any[1] ? 0 : n_list};
  for (;;) {
    int64_t tiles[3] = {0, 0, 0};
    for (int big = 0; big < 2; ++big) {
      ExpertList& list = big ? a.list : a.small;
      list.n = list.n_mid = 0;
      for (int32_t& i = at[big]; i < n_list && list.n < kListMax; ++i) {
        if (list_rows && (list_rows[i] < 1 || (list_rows[i] > kSmallRows) != (big != 0))) continue;
        if (list_rows && big)
          for (int by = 0; by < 3; ++by) tiles[by] += ceil_div(list_rows[i], 256 >> by);
        entry[list.n++] = {list_rows ? list_rows[i] : 0, expert_list[i]};
      }
      // the experts with most rows first: tiles of few rows, which take less time, fill the last round (777 tokens
      // of 64 experts as at tile_of: 65 us up instead of 72)
      if (big && list_rows)
        std::sort(entry, entry + list.n, [](const Entry& p, const Entry& q) { return p.rows > q.rows; });
      for (int i = 0; i < list.n; ++i) {
        list.expert[i] = (int16_t)entry[i].expert;
        list.slot[i] = slot_of[entry[i].expert];
      }
    }
    if (a.list.n + a.small.n == 0) return 0;
    // row counts unknown: sum ceil(n / rows) <= pairs / rows + the experts with more than kSmallRows rows
    if (!list_rows && a.list.n) {
      const int64_t most = pairs / (kSmallRows + 1);
      for (int by = 0; by < 3; ++by) tiles[by] = pairs / (256 >> by) + (a.list.n < most ? a.list.n : most);
    }
    const int rc = quantised ? launch_lists<true>(a, tiles, phases, cus, spare_cus, (hipStream_t)stream)
                             : launch_lists<false>(a, tiles, phases, cus, spare_cus, (hipStream_t)stream);
    if (rc) return rc;
  }
}
