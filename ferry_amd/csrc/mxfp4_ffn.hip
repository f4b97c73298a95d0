// Grouped SwiGLU expert FFN over MXFP4 cache slots.
//
// For each expert e with rows p in [starts[e], starts[e+1]):
//   x = in[rows[p]];  g = x Wg^T;  u = x Wu^T;  a = silu(g) * u;  y = a Wd^T;
//   out = bf16(y * w[rows[p], cols[p]])
// with cache[slot] = [codes of Wg (I x H) | Wu (I x H) | Wd (H x I), then their scales], the MXFP4 form
// of the bf16 cache row (mxfp4.hip).  Sums are fp32.  Two kinds of activations:
//  * bf16 (Q = false): x is bf16 and a is rounded to bf16, an operand of the bf16 matrix instruction.
//    The 4-bit weights become bf16 in registers, which is exact.
//  * MXFP4 (Q = true): x is codes and scales, and a is quantised from fp32 in the up epilogue, per 32
//    columns, as mxfp4_quantize does; both products run on the scaled 4-bit matrix instruction.
//
// A lane's 16-byte load of weight codes is one block of 32 along K with one scale.  In a chunk of 128
// along K, the lanes of row r take the blocks lane / 16 = 0..3: for the 4-bit instruction that is its
// operand layout, and for the bf16 one the four steps s of a chunk multiply the elements 8 s .. 8 s + 7
// of the blocks; the order along K inside a product is free as long as both operands share it.  So the
// weights go from the plain row-major rows straight to registers, with no LDS, shuffle or repacking.
#include "ffn_common.h"

#include <type_traits>

namespace ferry {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kSmallRows = 16;   // experts with at most this many rows run mx_small

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
  int32_t known;            // the listed experts' row counts were given
  ExpertList list;
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

// One workgroup: 16 NF weight rows (MODE 0: 8 NF columns of gate and of up; MODE 1: 16 NF hidden rows) x the
// expert's rows.  Its four wavefronts split K in units of 256, whose sums meet in LDS in wavefront order.
// Bound by the weight bytes: a wavefront brings up to kUnits units of its weights at once, by direct loads
// of whole cache lines (8 rows x 128 bytes) into LDS, from where it reads the operands (swizzled as in the
// tiles below); straight to registers in operand order, the lanes' 64 places of 16 bytes a load bound the
// kernel at 3 TB/s.  The rows' activations go to registers: only the lanes of rows that are there load.
constexpr int kUnits = 2;
__device__ __forceinline__ int swz_w16(int row) { return (row >> 1) & 7; }   // 16 consecutive rows

template <int MODE, bool Q, int NF>
__global__ __launch_bounds__(256) void mx_small(MxArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  constexpr int kRowsW = 16 * NF, kW = kRowsW * 128, kUnit = kW + kRowsW * 8;   // LDS of a unit: codes, scales
  const int li = blockIdx.y, bx = blockIdx.x;
  const int e = a.list.expert[li], slot = a.list.slot[li];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int64_t K = MODE == 0 ? a.H : a.I;
  const int chunks = (int)(K / 128), units = (chunks + 1) / 2;
  const int u0 = wave * units / 4, u1 = (wave + 1) * units / 4;
  const uint32_t lds0 = lds_addr(smem) + (uint32_t)(wave * min(kUnits, (units + 3) / 4) * kUnit);

  const Weights wp0 = weights_at<MODE>(a, slot, 0, MODE == 0 ? bx * (8 * NF) : bx * (16 * NF));
  const Weights wp1 = MODE == 0 ? weights_at<MODE>(a, slot, 1, bx * (8 * NF)) : wp0;
  u32x2 sv[kUnits];
  auto load_w = [&](int u, int b) {
    const uint32_t dst = lds0 + (uint32_t)(b * kUnit);
    const bool tail = 2 * u + 1 >= chunks;   // half a unit: its other half is read again, not multiplied
#pragma unroll
    for (int j = 0; j < 2 * NF; ++j) {
      const int t = 8 * j + (lane >> 3), part = MODE == 0 ? j / NF : 0;
      const int piece = (lane & 7) ^ swz_w16(t);
      const uint32_t off = (uint32_t)(t - part * 8 * NF) * (uint32_t)(K / 2) + (uint32_t)((tail ? piece & 3 : piece) * 16);
      dma16(reinterpret_cast<const char*>(uniform_ptr((part ? wp1.codes : wp0.codes) + u * 128)), off,
            dst + (uint32_t)(j * 1024));
    }
    const int part = MODE == 0 && lane >= 8 * NF;
    const uint8_t* sp = (part ? wp1.scales : wp0.scales) + (int64_t)(lane - part * 8 * NF) * (K / 32) + u * 8;
    if (lane < kRowsW) {
      if (tail) __builtin_memcpy(&sv[b], sp, 4);
      else __builtin_memcpy(&sv[b], sp, 8);
    }
  };
  // the first units' weights do not depend on the expert's rows: where those are known to be 1 to 16, their
  // loads go first
  if (a.known)
#pragma unroll
    for (int b = 0; b < kUnits; ++b)
      if (u0 + b < u1) load_w(u0 + b, b);
  const int64_t start = a.starts[e];
  const int64_t n = a.starts[e + 1] - start;
  if (n < 1 || n > kSmallRows) {
    wait_cnt<0>();
    return;
  }
  const bool live = r < n;
  const int64_t p = start + (live ? r : 0);
  const int64_t src = MODE == 0 ? a.rows[p] : p;
  const uint8_t* xp = MODE == 0 ? a.x : a.act;
  const uint8_t* xs = MODE == 0 ? a.x_scales : a.act_scales;
  xp += Q ? src * (K / 2) + q * 16 : src * K * 2 + q * 64;
  if (Q) xs += src * (K / 32) + q;
  floatx4 acc[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) acc[f] = floatx4{0, 0, 0, 0};
  for (int u = u0; u < u1; u += kUnits) {
    if (u > u0 || !a.known)
#pragma unroll
      for (int b = 0; b < kUnits; ++b)
        if (u + b < u1) load_w(u + b, b);
    constexpr int XL = Q ? 1 : 4;   // 16-byte loads of a lane and chunk
    u32x4 xv[kUnits][2][XL] = {};
    uint32_t xb[kUnits][2] = {};
    if (live)
#pragma unroll
      for (int b = 0; b < kUnits; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int c = 2 * (u + b) + j;
          if (u + b < u1 && c < chunks) {
#pragma unroll
            for (int s = 0; s < XL; ++s) xv[b][j][s] = *(const u32x4*)(xp + (int64_t)c * (Q ? 64 : 256) + s * 16);
            if (Q) xb[b][j] = xs[c * 4];
          }
        }
#pragma unroll
    for (int b = 0; b < kUnits; ++b)
      if (u + b < u1 && lane < kRowsW)
        *reinterpret_cast<__attribute__((address_space(3))) u32x2*>(
            (uintptr_t)(lds0 + (uint32_t)(b * kUnit + kW + lane * 8))) = sv[b];
    wait_cnt<0>();   // the wavefront's own LDS: no barrier
#pragma unroll
    for (int b = 0; b < kUnits; ++b) {
      if (u + b >= u1) break;
      const uint32_t at = lds0 + (uint32_t)(b * kUnit);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (2 * (u + b) + j >= chunks) break;
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
    }
  }
  __syncthreads();   // the weights' LDS becomes that of the sums
  floatx4(*part)[NF][64] = reinterpret_cast<floatx4(*)[NF][64]>(smem);
#pragma unroll
  for (int f = 0; f < NF; ++f) part[wave][f][lane] = acc[f];
  __syncthreads();
  // lane l of a tile holds the columns (l / 16) * 4 + i of row l % 16
  auto sum = [&](int f) {
    floatx4 v = part[0][f][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) v += part[w][f][lane];
    return v;
  };
  if constexpr (MODE == 0) {
    if constexpr (Q) {
      static_assert(NF == 4);   // a block of 32 columns
      if (wave != 0) return;
      float v[8];   // columns 16 (i / 4) + 4 q + i % 4
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const floatx4 g = sum(b), u = sum(2 + b);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * b + i] = silu_mul(g[i], u[i]);
      }
      const int byte = block_scale(v);
      const uint32_t c = block_codes(v, byte);
      if (live) {
        uint8_t* o = a.act + p * (a.I / 2) + bx * 16 + q * 2;
        *(uint16_t*)o = (uint16_t)c;
        *(uint16_t*)(o + 8) = (uint16_t)(c >> 16);
        if (q == 0) a.act_scales[p * (a.I / 32) + bx] = (uint8_t)byte;
      }
    } else {
      if (wave >= NF / 2) return;
      const floatx4 g = sum(wave), u = sum(NF / 2 + wave);
      u32x2 y;
#pragma unroll
      for (int i = 0; i < 4; i += 2) y[i / 2] = pk_bf16(silu_mul(g[i], u[i]), silu_mul(g[i + 1], u[i + 1]));
      if (live) *(u32x2*)(a.act + (p * a.I + bx * (8 * NF) + wave * 16 + q * 4) * 2) = y;
    }
  } else {
    if (wave >= NF) return;
    const floatx4 y = sum(wave);
    if (live) {
      const int64_t t = a.rows[p] * a.k + a.cols[p];
      const float wt = bf16_to_f32(a.w[t]);
      const int64_t o = a.out_mode == 0 ? t : p;
      *(u32x2*)(a.out + o * a.H + bx * (16 * NF) + wave * 16 + q * 4) =
          u32x2{pk_bf16(y[0] * wt, y[1] * wt), pk_bf16(y[2] * wt, y[3] * wt)};
    }
  }
}

template <int MODE, bool Q, int NF>
int small_launch(const MxArgs& a, hipStream_t s) {
  const int64_t K = MODE == 0 ? a.H : a.I, units = ceil_div(K, 256);
  const dim3 g((unsigned)(MODE == 0 ? a.I / (8 * NF) : a.H / (16 * NF)), (unsigned)a.list.n);
  const int64_t bytes = 4 * (units > 4 ? kUnits : 1) * (16 * NF * 136), sums = 4 * NF * 1024;
  launch(MODE == 0 ? "mx_small_up" : "mx_small_down", mx_small<MODE, Q, NF>, g, dim3(256),
         (uint32_t)(bytes > sums ? bytes : sums), s, a);
  FERRY_LAUNCHED("mx_small");
  return 0;
}

// =============================================================================================
// Larger experts: tiles of TM rows x TN weight rows
// =============================================================================================

// WM x WN wavefronts, each MI x 4 tiles of 16 rows x 16 weight rows.  Activations and weights are staged in
// LDS by direct loads, in rows of 128 bytes (whole cache lines, eight lanes a row): 256 along K of 4-bit
// values (a stage), 64 of bf16 (four steps to a stage).  Loading the weights to registers in operand order
// instead takes no LDS, but its lanes touch 64 places of 16 bytes: address processing then bounds the kernel
// (5 us for 128 along K, whatever the products).  Two buffers each, the loads one stage or step ahead of
// the products, across tiles too: the last ones of a tile load the first of the next, whose rows are looked
// up meanwhile.  A row's 16-byte pieces are stored at slot piece ^ swizzle(row), so that the 16 rows that a
// quarter of a wavefront reads lie on 16 different 16-byte bank groups.
// Rows of a tile that hold no row of the expert are neither loaded nor multiplied, in steps of a quarter.
// (bf16) The weights of a step are read before the barrier that its rows wait for.
// MODE 0: of a wavefront's four weight tiles, two are gate rows and two the up rows of the same 32 columns.
// The weight rows of the two tiles c of 32 columns interleave in groups of four, 8 g + 4 c + [0, 4):
// a lane then holds 8 consecutive output columns of one row.
__device__ __forceinline__ int swz_x(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int swz_w(int row) { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); }

template <int MODE, bool Q, int WM, int WN, int MI>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(WM * WN / 4, WM * WN / 4)))
void mx_tiled(MxArgs a) {
  constexpr int NI = 4, W = WM * WN, TM = 16 * WM * MI, TN = 16 * NI * WN;
  constexpr int COLS = MODE == 0 ? TN / 2 : TN;          // output columns of a tile
  constexpr int kX = TM * 128, kW = TN * 128;            // bytes of a buffer
  constexpr int LX = kX / (1024 * W), LW = kW / (1024 * W);   // direct loads of a wavefront for one
  constexpr int kXS = Q ? TM * 8 : 0, kWS = TN * 8;      // scale bytes of a stage
  constexpr int kScaleRows = TN + (Q ? TM : 0);
  static_assert(LX == 4 && TM == 32 * W && LW >= 1 && kScaleRows <= 64 * W && TM <= 64 * W && MI % 4 == 0);
  __shared__ TileTable tt;
  __shared__ __attribute__((aligned(1024))) char smem[2 * (kX + kW + kXS + kWS)];
  // per tile row, two sets taken in turn: the token, and for MODE 1 the slot index, the output row and the
  // routing weight (bf16 bits)
  __shared__ __attribute__((aligned(256))) int32_t row_s[2][TM], col_s[MODE == 1 ? 2 : 1][MODE == 1 ? TM : 1];
  __shared__ __attribute__((aligned(256))) int32_t orow_s[MODE == 1 ? 2 : 1][MODE == 1 ? TM : 1],
      wt_s[MODE == 1 ? 2 : 1][MODE == 1 ? TM : 1];
  build_tile_table<TM, kSmallRows>(a, tt);
  const int64_t K = MODE == 0 ? a.H : a.I;
  const int ntn = (int)((MODE == 0 ? a.I : a.H) / COLS);
  const int total = __builtin_amdgcn_readfirstlane(tt.total) * ntn;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int r = lane & 15, q = lane >> 4;
  const int chunks = (int)(K / 128), stages = (chunks + 1) / 2;
  const uint32_t smem0 = lds_addr(smem);
  const uint32_t wbuf = smem0 + 2 * kX, xsbuf = wbuf + 2 * kW, wsbuf = xsbuf + 2 * kXS;
  const char* const xbase = reinterpret_cast<const char*>(MODE == 0 ? a.x : a.act);
  const uint8_t* const xsbase = MODE == 0 ? a.x_scales : a.act_scales;

  // fragment reads: addresses of tile 0, the others at constant offsets
  const int xrow = 16 * wm + r;
  const int wrow = (MODE == 0 ? wn * 32 : wn * 64) + 8 * (r >> 2) + (r & 3);
  const uint32_t xa = smem0 + (uint32_t)(xrow * 128 + (((Q ? q : 2 * q) ^ swz_x(xrow)) << 4));
  const uint32_t wa = wbuf + (uint32_t)(wrow * 128 + (((Q ? q : q >> 1) ^ swz_w(wrow)) << 4) + (Q ? 0 : (q & 1) * 8));
  constexpr int kXTile = 16 * WM * 128;
  auto wtile = [](int f) { return (f >> 1) * (MODE == 0 ? TN / 2 : 32) + (f & 1) * 4; };   // in rows

  struct Tile {
    int64_t row0;        // grouped row of the tile's first row
    int vrows, nt, slot;
  };
  auto locate = [&](int tile) {
    Tile t;
    const int mt = tile / ntn;
    t.nt = tile - mt * ntn;
    const int li = __builtin_amdgcn_readfirstlane(find_entry(tt, mt));
    const int m0 = (mt - __builtin_amdgcn_readfirstlane(tt.cum[li])) * TM;
    t.row0 = uniform64(tt.start[li]) + m0;
    t.vrows = __builtin_amdgcn_readfirstlane(tt.rows[li]) - m0;   // > 0
    t.slot = a.list.slot[li];
    return t;
  };
  // the tile rows' indices (low words; rows past the last: the first row's) into set p, direct loads
  auto load_rows = [&](const Tile& t, int p) {
    if (wave < TM / 64) {
      const int v = 64 * wave + lane;
      const uint32_t off = (uint32_t)((v < t.vrows ? v : 0) * 8);
      dma4(reinterpret_cast<const char*>(uniform_ptr(a.rows + t.row0)), off, lds_addr(row_s[p]) + 256 * wave);
      if constexpr (MODE == 1)
        dma4(reinterpret_cast<const char*>(uniform_ptr(a.cols + t.row0)), off, lds_addr(col_s[p]) + 256 * wave);
    }
  };

  // The tiles whose activations and weights are being loaded.  Direct load j of a wavefront moves 8 rows, lane / 8 of them,
  // its lane % 8 the piece (lane % 8) ^ swizzle: rows 64 j .. of the activations over all wavefronts (W = 8),
  // so that a tile of few rows takes the first loads only.
  const int r8 = lane >> 3, slot8 = lane & 7;
  auto xload_row = [&](int j) { return 8 * (W * j + wave) + r8; };
  uint32_t xoff[LX], woff[LW], sdst;
  const char* wbase[LW];
  const uint8_t* sp = nullptr;   // this thread's row of scales: a weight row, or (Q) an activation row
  int xloads = LX;
  if (tid < TN) sdst = wsbuf + (uint32_t)(tid * 8);
  else sdst = xsbuf + (uint32_t)((tid - TN) * 8);
  auto aim_x = [&](const Tile& t, int p) {
    auto src_row = [&](int v) {
      return MODE == 0 ? (uint32_t)row_s[p][v] : (uint32_t)(t.row0 + (v < t.vrows ? v : 0));
    };
    xloads = t.vrows > TM / 4 * 3 ? 4 : (t.vrows > TM / 2 ? 3 : (t.vrows > TM / 4 ? 2 : 1));
#pragma unroll
    for (int j = 0; j < LX; ++j) {
      const int v = xload_row(j);
      xoff[j] = src_row(v) * (uint32_t)(Q ? K / 2 : K * 2) + (uint32_t)((slot8 ^ swz_x(v)) * 16);
    }
    if (Q && tid >= TN && tid < kScaleRows) sp = xsbase + (int64_t)src_row(tid - TN) * (K / 32);
  };
  auto aim_w = [&](const Tile& t) {
    const Weights m0 = weights_at<MODE>(a, t.slot, 0, t.nt * COLS);
    const Weights m1 = MODE == 0 ? weights_at<MODE>(a, t.slot, 1, t.nt * COLS) : m0;
#pragma unroll
    for (int j = 0; j < LW; ++j) {
      const int t0 = 8 * (wave * LW + j), part = MODE == 0 ? t0 / (TN / 2) : 0;
      wbase[j] = reinterpret_cast<const char*>(uniform_ptr(part ? m1.codes : m0.codes));
      woff[j] = (uint32_t)(t0 - part * (TN / 2) + r8) * (uint32_t)(K / 2) + (uint32_t)((slot8 ^ swz_w(t0 + r8)) * 16);
    }
    if (tid < TN) {
      const int part = MODE == 0 ? tid / (TN / 2) : 0;
      sp = (part ? m1.scales : m0.scales) + (int64_t)(tid - part * (TN / 2)) * (K / 32);
    }
  };
  u32x2 sv = {0, 0};
  auto load_s = [&](int st) {
    if (tid < kScaleRows) {
      if (2 * st + 1 < chunks) __builtin_memcpy(&sv, sp + st * 8, 8);
      else __builtin_memcpy(&sv, sp + st * 8, 4);
    }
  };
  auto store_s = [&](int b) {
    if (tid < kScaleRows)
      *reinterpret_cast<__attribute__((address_space(3))) u32x2*>((uintptr_t)(sdst + (uint32_t)(b * (tid < TN ? kWS : kXS)))) = sv;
  };
  // Where the number of chunks is odd, the last stage's rows of 4-bit values end in its middle: the lanes of
  // the second half read the first half again (it is not multiplied).
  auto back = [&](int piece) { return (uint32_t)((piece & 4) << 4); };
  auto load_x = [&](int n, int b) {   // Q: stage n; bf16: step n
    const uint32_t dst = smem0 + (uint32_t)(b * kX + wave * 1024);
#pragma unroll
    for (int j = 0; j < LX; ++j)
      if (j < xloads) {
        const uint32_t tail = Q && 2 * n + 1 >= chunks ? back(slot8 ^ swz_x(xload_row(j))) : 0u;
        dma16(xbase + (int64_t)n * 128, xoff[j] - tail, dst + (uint32_t)(W * j * 1024));
      }
  };
  auto load_w = [&](int st, int b) {
#pragma unroll
    for (int j = 0; j < LW; ++j) {
      const uint32_t tail = 2 * st + 1 >= chunks ? back(slot8 ^ swz_w(8 * (wave * LW + j) + r8)) : 0u;
      dma16(wbase[j] + (int64_t)st * 128, woff[j] - tail, wbuf + (uint32_t)(b * kW + (wave * LW + j) * 1024));
    }
  };

  // XCD-aware order: workgroup b runs on XCD b % 8, whose workgroups take a contiguous run of tiles; tiles of
  // one expert follow each other, columns fastest, and share their rows and weights in that XCD's L2.
  const int per_xcd = gridDim.x % 8 == 0 ? (int)gridDim.x / 8 : 0;
  const int first = per_xcd ? (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8) : (int)blockIdx.x;
  if (first >= total) return;
  Tile cur = locate(first);
  load_rows(cur, 0);
  wait_cnt<0>();
  wg_barrier();
  aim_x(cur, 0);
  aim_w(cur);
  load_s(0);
  load_w(0, 0);
  load_x(0, 0);
  store_s(0);
  wait_cnt<0>();
  wg_barrier();
  int set = 0, wb = 0;   // set of row tables; buffer of the present stage (Q: of its activations too)

  // bf16: the weights' codes of the next step, their scales of its chunk
  u32x2 wr[NI];
  uint32_t ws[NI];
  auto read_w = [&](uint32_t at) {
#pragma unroll
    for (int f = 0; f < NI; ++f) wr[f] = lds_get<lds_u32x2>(at + (uint32_t)(wtile(f) * 128));
  };
  auto read_s = [&](uint32_t at) {
#pragma unroll
    for (int f = 0; f < NI; ++f) ws[f] = lds_get<lds_u32>(at + (uint32_t)((wrow + wtile(f)) * 8));
  };
  if constexpr (!Q) {
    read_w(wa);
    read_s(wsbuf);
  }
  for (int tile = first; tile < total; tile += gridDim.x, set ^= 1) {
    // the tile after this one; after the last tile its own first stage is loaded again
    const bool more = tile + (int)gridDim.x < total;
    const Tile next = more ? locate(tile + gridDim.x) : cur;
    load_rows(next, set ^ 1);
    if constexpr (MODE == 1) {
      // output row and routing weight of tile row tid, in LDS before the epilogue reads them
      if (wave < TM / 64) {
        const int64_t tj = (int64_t)row_s[set][tid] * a.k + col_s[set][tid];
        dma2(reinterpret_cast<const char*>(a.w), (uint32_t)(tj * 2), lds_addr(wt_s[set]) + 256 * wave);
        orow_s[set][tid] = a.out_mode == 0 ? (int32_t)tj : (int32_t)(cur.row0 + (tid < cur.vrows ? tid : 0));
      }
    }
    floatx4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int f = 0; f < NI; ++f) acc[i][f] = floatx4{0, 0, 0, 0};
    // In the last stage (bf16 activations: step) the loads turn to the next tile, whose row indices may still
    // be on their way where it is the only one.
    auto turn_x = [&]() {
      if (stages == 1) {
        wait_cnt<0>();
        wg_barrier();
      }
      aim_x(next, set ^ 1);
    };
    // ROWS: tiles of 16 rows of a wavefront that are multiplied; the others hold no row of the expert
    auto loop = [&](auto rows) {
      constexpr int ROWS = decltype(rows)::value;
      if constexpr (Q) {
        for (int st = 0; st < stages; ++st, wb ^= 1) {
          const uint32_t xb = xa + (uint32_t)(wb * kX), wbb = wa + (uint32_t)(wb * kW);
          const uint32_t xsb = xsbuf + (uint32_t)(wb * kXS + xrow * 8), wsb = wsbuf + (uint32_t)(wb * kWS + wrow * 8);
          u32x4 xn[2], wf[NI];
          uint32_t xsn[2], wsf[NI];
          auto read_x = [&](int j, int i) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              xn[v] = lds_get<lds_u32x4>((xb ^ (uint32_t)(j << 6)) + (uint32_t)(kXTile * (i + v)));
              xsn[v] = lds_get<lds_u32>(xsb + (uint32_t)(16 * WM * 8 * (i + v) + 4 * j));
            }
          };
          auto read_wq = [&](int j) {
#pragma unroll
            for (int f = 0; f < NI; ++f) {
              wf[f] = lds_get<lds_u32x4>((wbb ^ (uint32_t)(j << 6)) + (uint32_t)(wtile(f) * 128));
              wsf[f] = lds_get<lds_u32>(wsb + (uint32_t)(wtile(f) * 8 + 4 * j));
            }
          };
          read_wq(0);
          read_x(0, 0);
          const bool last = st + 1 == stages;
          if (last) {
            turn_x();
            aim_w(next);
          }
          const int ls = last ? 0 : st + 1;
          load_s(ls);
          load_w(ls, wb ^ 1);
          load_x(ls, wb ^ 1);
          const bool two = 2 * st + 1 < chunks;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (j == 1 && !two) break;
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
                read_wq(1);
              }
#pragma unroll
              for (int f = 0; f < NI; ++f) acc[i][f] = mma_fp4(cw[f], cs[f], x0, s0, acc[i][f]);
#pragma unroll
              for (int f = 0; f < NI; ++f) acc[i + 1][f] = mma_fp4(cw[f], cs[f], x1, s1, acc[i + 1][f]);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
          store_s(wb ^ 1);
          wait_cnt<0>();   // the next stage's loads have landed, this one's fragments are read
          wg_barrier();
        }
      } else {
        for (int c = 0; c < chunks; ++c) {
          const bool first_half = (c & 1) == 0, last = c + 1 == chunks;
          const bool stage_end = !first_half || last;   // the next chunk lies in the other buffer
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t xb = xa, wat = wa;   // computed here, not kept in registers through the loop
            asm volatile("" : "+v"(xb), "+v"(wat));
            xb += (uint32_t)(h * kX);
            bf16x8 xr[3];
            auto read = [&](int m) {
              xr[m % 3] = lds_read16((xb ^ (uint32_t)((m / ROWS) << 4)) + (uint32_t)(kXTile * (m % ROWS)));
            };
            read(0);
            read(1);
            // the first 32 along K are decoded while the first fragments are on their way, the second 32
            // between the products of the first
            u32x4 wv[2][NI];
            uint32_t c1[NI];
            float sc[NI];
            auto decode = [&](uint32_t v, int s, int part) {   // half of a weight tile's 8 elements a lane
              const int f = part >> 1, half = part & 1;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const bf16x2 d = half ? (j ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc[f], 3)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc[f], 2))
                                      : (j ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc[f], 1)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc[f], 0));
                wv[s][f][2 * half + j] = __builtin_bit_cast(uint32_t, d);
              }
            };
#pragma unroll
            for (int f = 0; f < NI; ++f)
              c1[f] = wr[f][1], sc[f] = scale_of(__builtin_amdgcn_ubfe(ws[f], 16 * h + 8 * (q >> 1), 8));
#pragma unroll
            for (int part = 0; part < 2 * NI; ++part) decode(wr[part >> 1][0], 0, part);
            __builtin_amdgcn_sched_barrier(0);
            if (h == 0) {
              if (first_half) {   // the next stage's weights: there one step later
                const bool final_stage = c + 2 >= chunks;
                if (final_stage) aim_w(next);
                load_s(final_stage ? 0 : c / 2 + 1);
                load_w(final_stage ? 0 : c / 2 + 1, wb ^ 1);
              }
              load_x(2 * c + 1, 1);
              read_w((wat + (uint32_t)(wb * kW)) ^ (uint32_t)((c & 1) << 6) ^ 32u);
            } else {
              if (last) turn_x();
              load_x(last ? 0 : 2 * c + 2, 0);
              if (stage_end) wb ^= 1;
              read_w((wat + (uint32_t)(wb * kW)) ^ (uint32_t)(stage_end ? 0 : 64));
              read_s(wsbuf + (uint32_t)(wb * kWS + (stage_end ? 0 : 4)));
            }
#pragma unroll
            for (int m = 0; m < 2 * ROWS; ++m) {
              const int s = m / ROWS, i = m % ROWS;
              if (m + 2 < 2 * ROWS) read(m + 2);
              if (s == 0)
#pragma unroll
                for (int part = i * 2 * NI / ROWS; part < (i + 1) * 2 * NI / ROWS; ++part) decode(c1[part >> 1], 1, part);
#pragma unroll
              for (int f = 0; f < NI; ++f)
                acc[i][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[s][f]), xr[m % 3],
                                                                   acc[i][f], 0, 0, 0);
              __builtin_amdgcn_sched_barrier(0);
            }
            if (h == 0 && first_half) store_s(wb ^ 1);
            wait_cnt<0>();
            wg_barrier();
          }
        }
      }
    };
    // rows 16 (WM i + wm) .. + 16 are tile i of wavefront row wm: the tile's rows in steps of a quarter
    if (cur.vrows > TM / 4 * 3) loop(std::integral_constant<int, MI>{});
    else if (cur.vrows > TM / 2) loop(std::integral_constant<int, MI / 4 * 3>{});
    else if (cur.vrows > TM / 4) loop(std::integral_constant<int, MI / 2>{});
    else loop(std::integral_constant<int, MI / 4>{});
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int t = 16 * (WM * i + wm) + r;
      const bool live = t < cur.vrows;
      if constexpr (MODE == 0) {
        float v[8];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[4 * c + j] = silu_mul(acc[i][c][j], acc[i][2 + c][j]);
        const int64_t col = cur.nt * COLS + wn * 32;
        if constexpr (Q) {
          const int byte = block_scale(v);
          const uint32_t c = block_codes(v, byte);
          if (live) {
            *(uint32_t*)(a.act + (cur.row0 + t) * (a.I / 2) + col / 2 + q * 4) = c;
            if (q == 0) a.act_scales[(cur.row0 + t) * (a.I / 32) + col / 32] = (uint8_t)byte;
          }
        } else if (live) {
          *(u32x4*)(a.act + ((cur.row0 + t) * a.I + col + q * 8) * 2) =
              u32x4{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7])};
        }
      } else if (live) {
        const float wt = __uint_as_float((uint32_t)wt_s[set][t] << 16);
        bf16_t* const o = a.out + (int64_t)orow_s[set][t] * a.H + cur.nt * COLS + wn * 64 + q * 8;
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
    cur = next;
  }
}

int device_cus(int* cus) {
  int dev = 0;
  FERRY_HIP(hipGetDevice(&dev));
  FERRY_HIP(hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev));
  if (*cus <= 0) *cus = 256;
  return 0;
}

// The launches of one list in one kind of activations; tiles: row tiles of 256 rows of the experts with more
// than kSmallRows rows (an upper bound).
template <bool Q>
int launch_list(const MxArgs& a, bool small, int64_t tiles, int32_t phases, int64_t cus, hipStream_t s) {
  for (int mode = 0; mode < 2; ++mode) {
    if (!(phases & (1 << mode))) continue;
    if (small)
      if (const int rc = mode == 0 ? small_launch<0, Q, Q ? 4 : 2>(a, s) : small_launch<1, Q, 4>(a, s)) return rc;
    if (tiles) {
      const int64_t t = tiles * (mode == 0 ? a.I / 128 : a.H / 256);
      launch(mode == 0 ? "mx_tiled_up" : "mx_tiled_down", mode == 0 ? mx_tiled<0, Q, 2, 4, 8> : mx_tiled<1, Q, 2, 4, 8>,
             dim3((unsigned)(t < cus ? t : cus)), dim3(512), 0, s, a);
      FERRY_LAUNCHED("mx_tiled");
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
  FERRY_CHECK_ARG(topk >= 1 && rows_in >= 0 && n_list >= 0 && max_rows_per_expert >= 0, "bad sizes");
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
  if (n_list == 0 || rows_in == 0) return 0;
  FERRY_CHECK_ARG(cache && x && w_sorted && starts && rows && cols && expert_list && slot_of && act && out,
                  "null pointer argument");
  FERRY_CHECK_ARG(((uintptr_t)cache | (uintptr_t)x | (uintptr_t)act | (uintptr_t)out) % 16 == 0,
                  "cache, x, act and out must be 16-byte aligned");
  FERRY_CHECK_ARG((uintptr_t)x_scales % 4 == 0, "x_scales must be 4-byte aligned");
  for (int32_t i = 0; i < n_list; ++i) {
    const int32_t e = expert_list[i];
    FERRY_CHECK_ARG(e >= 0 && e < experts, "expert_list[%d] = %d out of range", i, e);
    const int32_t s = slot_of[e];
    FERRY_CHECK_ARG(s >= 0 && s < cache_rows, "expert %d is not cached (slot %d)", e, s);
    if (list_rows)
      FERRY_CHECK_ARG(list_rows[i] >= min_rows_per_expert && list_rows[i] <= max_rows_per_expert,
                      "list_rows[%d] = %d outside [min_rows_per_expert, max_rows_per_expert]", i,
                      list_rows[i]);
  }
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  if (cus > 2 * spare_cus) cus -= spare_cus;
  const bool quantised = x_scales != nullptr;
  const int64_t pairs = rows_in * topk;
  MxArgs a;
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
  a.list.n_mid = 0;
  // one pass over the small experts, one over the others; without row counts every expert is in both, and
  // the kernels pass over those of the other kind by the device's starts
  for (int big = 0; big < 2; ++big) {
    if (big ? max_rows_per_expert <= kSmallRows : min_rows_per_expert > kSmallRows) continue;
    int64_t tiles = 0;
    a.list.n = 0;
    auto flush = [&]() {
      if (a.list.n == 0) return 0;
      // row counts unknown: sum ceil(n / 256) <= pairs / 256 + the experts with more than kSmallRows rows
      if (big && !list_rows) tiles = pairs / 256 + (a.list.n < pairs / (kSmallRows + 1) + 1 ? a.list.n : pairs / (kSmallRows + 1) + 1);
      const int rc = quantised ? launch_list<true>(a, !big, tiles, phases, cus, (hipStream_t)stream)
                               : launch_list<false>(a, !big, tiles, phases, cus, (hipStream_t)stream);
      a.list.n = 0;
      tiles = 0;
      return rc;
    };
    for (int32_t i = 0; i < n_list; ++i) {
      if (list_rows) {
        if (list_rows[i] < 1 || (list_rows[i] > kSmallRows) != (big != 0)) continue;
        if (big) tiles += ceil_div(list_rows[i], 256);
      }
      a.list.expert[a.list.n] = (int16_t)expert_list[i];
      a.list.slot[a.list.n++] = slot_of[expert_list[i]];
      if (a.list.n == kListMax)
        if (const int rc = flush()) return rc;
    }
    if (const int rc = flush()) return rc;
  }
  return 0;
}
