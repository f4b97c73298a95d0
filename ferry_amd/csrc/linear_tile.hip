// The linear products on whole tiles: rows at multiples of 16 bytes, sizes of multiples of 8.
#include "linear_plan.h"
#include "linear_stream.h"
#include "linear_tile.h"

#include <algorithm>
#include <type_traits>

namespace ferry {
namespace lin {
namespace {

// =============================================================================================
// 256 x 256 tiles
// =============================================================================================
//
// A workgroup of eight wavefronts, two per SIMD, computes 256 x 256 outputs; bound by the matrix cores.  The
// schedule is that of the expert FFN's large tiles: a stage holds 64 of the contraction, each operand as two
// halves of 128 indices (16 KiB); wavefront (wm, wn) = (w / 4, w % 4) computes in each quadrant (A half, B
// half) the indices 32 i + 16 wm + [0, 16) of A (i < 4) by 32 wn + [0, 32) of B.
//
//   phase            1        2        3        4
//   reads            A0(k)    B1(k)    A1(k)    B0(k+1)
//   loads            B0(k+2)  A0(k+2)  B1(k+2)  A1(k+2)    (into the half read one phase before)
//   multiplies       A0 B0    A0 B1    A1 B0    A1 B1
//
// Each phase is a memory and a matrix segment with a barrier after each; the wavefronts wm = 1 run one
// segment behind, so that one of a SIMD's two multiplies while the other reads and loads.  A half is loaded
// seven phases before it is read, two loads a wavefront and phase, so "at most 12 outstanding" says that the
// half read next has landed.  The last two stages of a tile load the first two of the next.
//
// Loads are buffer loads straight to LDS: whatever lies behind an operand's last row or a group's end reads
// as 0, so ragged sizes cost no test in the loop.  A contraction that is no multiple of 64 ends inside the
// rows of an operand staged by index; there the lanes whose chunk lies behind it get an offset behind the
// buffer before the last stage.
//
// The B indices belong to the products' first operand, so a lane holds four consecutive output columns of
// one row.  Two tiles of 16 columns give 8 and one 16-byte store: of an operand staged by index, whose
// fragments take any rows, the columns 8 g + 4 c + [0, 4) of tile c; of one staged by c, whose fragments take
// 16 consecutive ones without bank conflicts, by an exchange between neighbouring rows of lanes at the end.
constexpr int kHalf = 128 * 128;   // bytes

template <typename T, int MODE, bool GATHER, int ACT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void tile256(Args a) {
  constexpr bool XA = MODE == kDw, XB = MODE != kFwd, RAG = MODE != kDw;
  constexpr bool GA = GATHER && MODE == kFwd, GB = GATHER && MODE == kDw;
  __shared__ Table tt;
  __shared__ typename Tiles<MODE, GATHER, 256, 256>::Store places;
  __shared__ __attribute__((aligned(1024))) char smem[8 * kHalf];
  // GA: the rows of x of a tile's rows, two tiles in turn.  GB: those of 8 stages, each wavefront its own 8
  // rows of a stage: sets 0 and 1 in turn, 2 and 3 for the first 8 stages of a tile.  Low and high words.
  __shared__ __attribute__((aligned(256))) uint32_t row_s[GA ? 2 : (GB ? 4 : 1)][2][GA ? 256 : (GB ? 512 : 1)];
  __shared__ __attribute__((aligned(256))) uint32_t bias_s[MODE == kFwd ? 2 : 1][MODE == kFwd ? 128 : 1];   // of the tile's columns, in turn
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  build_table<RAG>(a, tt, RAG ? 256 : (int)ceil_div(a.I, 256));
  if (RAG && a.zero_rest) zero_rest(a, tt.first, tt.last);
  Tiles<MODE, GATHER, 256, 256> tiles(a, tt, places);
  if (!tiles.next()) return;
  const int wm = wave >> 2, wn = wave & 3;
  const int j16 = lane & 15, g4 = lane >> 4;
  const uint32_t smem0 = lds_at(smem);

  // fragment reads.  Staged by index: one address for each K step, tiles at constant distances.  By c: one
  // for each tile (the swizzle exchanges tiles), K steps and halves of a fragment at constant distances.
  uint32_t a_addr[XA ? 4 : 2], b_addr[2];
  if constexpr (XA) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a_addr[i] = smem0 + frag_across<128>(32 * i + 16 * wm, 0, 0);
  } else {
    const int r = 16 * wm + j16;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) a_addr[ks] = smem0 + (uint32_t)(r * 128 + (((4 * ks + g4) ^ swz_direct(r)) << 4));
  }
  if constexpr (XB) {
#pragma unroll
    for (int c = 0; c < 2; ++c) b_addr[c] = smem0 + 4 * kHalf + frag_across<128>(32 * wn + 16 * c, 0, 0);
  } else {
    const int r = 32 * wn + 8 * (j16 >> 2) + (j16 & 3);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      b_addr[ks] = smem0 + 4 * kHalf + (uint32_t)(r * 128 + (((4 * ks + g4) ^ swz_pair(r)) << 4));
  }

  const uint32_t lda2 = (uint32_t)a.lda * 2, ldb2 = (uint32_t)a.ldb * 2;
  const uint32_t a_step = XA ? 64 * lda2 : 128, b_step = XB ? (GB ? 0 : 64 * ldb2) : 128;

  // The load stream: the tile whose stages are being loaded.  Staged by index: a wavefront's rows 16 wave +
  // 8 q + lane / 8 of a half, place lane % 8.  By c: its rows 8 wave + 4 q + lane / 16, place lane % 16.
  u32x4 ra, rb;                  // buffers
  uint32_t sa = 0, sb = 0;       // the stage's offset in them
  uint32_t a_half, b_half;       // from half 0 to half 1
  int left = 0;                  // of the contraction, from the stage on
  const int64_t* idx = nullptr;  // GB: row numbers from the stage on
  uint32_t avo[GA ? 2 : 1][2], bvo[2];
  auto chunk_a = [&](int q) __attribute__((always_inline)) {
    return XA ? (lane & 15) ^ swz_across<128>(8 * wave + 4 * q + (lane >> 4))
              : (lane & 7) ^ swz_direct(16 * wave + 8 * q + (lane >> 3));
  };
  auto chunk_b = [&](int q) __attribute__((always_inline)) {
    return XB ? (lane & 15) ^ swz_across<128>(8 * wave + 4 * q + (lane >> 4))
              : (lane & 7) ^ swz_pair(16 * wave + 8 * q + (lane >> 3));
  };
  // GA: the row numbers of a tile's `n` rows into set p
  auto tile_rows = [&](const int64_t* at, int n, int p) __attribute__((always_inline)) {
    if (wave < 4) {
      const u32x4 r = buffer_at(at, (int64_t)(n < 256 ? n : 256) * 8);
      const uint32_t o = (uint32_t)(64 * wave + lane) * 8;
      load_lds4(r, o, lds_at(row_s[p][0]) + 256 * wave);
      load_lds4(r, o + 4, lds_at(row_s[p][1]) + 256 * wave);
    }
  };
  // GB: those of 8 stages, `n` c from `at` on, into set p
  auto stage8_rows = [&](const int64_t* at, int n, int p) __attribute__((always_inline)) {
    const u32x4 r = buffer_at(at, (int64_t)n * 8);
    const uint32_t o = (uint32_t)((lane >> 3) * 64 + 8 * wave + (lane & 7)) * 8;
    load_lds4(r, o, lds_at(row_s[p][0]) + 256 * wave);
    load_lds4(r, o + 4, lds_at(row_s[p][1]) + 256 * wave);
  };
  // the stream goes on with the tile t; GA: p its set of row numbers
  auto begin_tile = [&](const Tile& t, int p) __attribute__((always_inline)) {
    ra = t.a, rb = t.b, sa = sb = 0, left = t.nc;
    if constexpr (GB) idx = a.rows + t.p0;
    // a half without rows or columns loads the other's: what it gives is not stored
    a_half = half_offset(XA, t.rows, lda2);
    b_half = half_offset(XB, a.J - t.j0, ldb2);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t ca = (uint32_t)chunk_a(q) * 16, cb = (uint32_t)chunk_b(q) * 16;
      if constexpr (GA) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 128 * h + 16 * wave + 8 * q + (lane >> 3);
          const uint32_t x = row_s[p][0][r];
          const bool ok = r < t.rows && row_s[p][1][r] == 0 && x < (uint64_t)a.x_rows;
          avo[h][q] = ok ? x * lda2 + ca : kNowhere;
        }
      } else {
        avo[0][q] = (uint32_t)(XA ? 8 * wave + 4 * q + (lane >> 4) : 16 * wave + 8 * q + (lane >> 3)) * lda2 + ca;
      }
      if constexpr (!GB) bvo[q] = (uint32_t)(XB ? 8 * wave + 4 * q + (lane >> 4) : 16 * wave + 8 * q + (lane >> 3)) * ldb2 + cb;
    }
  };
  // before the stage k of the stream's tile is loaded; GB: p the tile's first set is 2 + p
  auto begin_stage = [&](int k, int p) __attribute__((always_inline)) {
    if (left <= 0) {   // not there: zeros
      ra[2] = rb[2] = 0;
      sa = sb = 0;
    } else if (!(XA && XB) && left < 64) {   // chunks behind the contraction's end lie nowhere
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (!XA && chunk_a(q) * 8 >= left) {
          avo[0][q] = kNowhere;
          if constexpr (GA) avo[1][q] = kNowhere;
        }
        if (!XB && chunk_b(q) * 8 >= left) bvo[q] = kNowhere;
      }
    }
    if constexpr (GB) {
      if ((k & 7) == 0) {
        if (left > 512) stage8_rows(idx + 512, left - 512, ((k >> 3) + 1) & 1);
        idx += 512;
      }
      const int set = k < 8 ? 2 + p : (k >> 3) & 1;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = 4 * q + (lane >> 4), at = 64 * wave + 8 * (k & 7) + r;
        const uint32_t x = row_s[set][0][at];
        const bool ok = 8 * wave + r < left && row_s[set][1][at] == 0 && x < (uint64_t)a.x_rows;
        bvo[q] = ok ? x * ldb2 + (uint32_t)chunk_b(q) * 16 : kNowhere;
      }
    }
  };
  auto end_stage = [&]() __attribute__((always_inline)) {
    left -= 64;
    sa += a_step;
    sb += b_step;
  };
  auto load_a = [&](int h, int slot) __attribute__((always_inline)) {
    const uint32_t dst = smem0 + (uint32_t)((2 * h + slot) * kHalf + 2048 * wave);
#pragma unroll
    for (int q = 0; q < 2; ++q) load_lds(ra, avo[GA ? h : 0][q], GA || h == 0 ? sa : sa + (left > 0 ? a_half : 0), dst + 1024 * q);
  };
  auto load_b = [&](int h, int slot) __attribute__((always_inline)) {
    const uint32_t dst = smem0 + (uint32_t)((4 + 2 * h + slot) * kHalf + 2048 * wave);
#pragma unroll
    for (int q = 0; q < 2; ++q) load_lds(rb, bvo[q], h == 0 ? sb : sb + (left > 0 ? b_half : 0), dst + 1024 * q);
  };

  s16x8 ft[4][2], fw[2][2][2];
  auto read_a = [&](auto hh, auto ss) __attribute__((always_inline)) {
    constexpr int off = (2 * decltype(hh)::value + decltype(ss)::value) * kHalf;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (XA)
          ft[i][ks] = read_across(a_addr[i] + (off + ks * 8192), a_addr[i] + (off + ks * 8192 + 1024));
        else
          ft[i][ks] = read_direct(a_addr[ks] + (off + i * 32 * 128));
      }
  };
  auto read_b = [&](auto hh, auto ss) __attribute__((always_inline)) {
    constexpr int H = decltype(hh)::value, off = (2 * H + decltype(ss)::value) * kHalf;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if constexpr (XB)
          fw[H][c][ks] = read_across(b_addr[c] + (off + ks * 8192), b_addr[c] + (off + ks * 8192 + 1024));
        else
          fw[H][c][ks] = read_direct(b_addr[ks] + (off + c * 4 * 128));
      }
  };

  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;

  int set = 0;   // GA: the set of the tile's row numbers; GB: its first set is 2 + set
  {
    const Tile t = tiles.tile();
    if constexpr (GA) tile_rows(a.rows + t.p0, t.rows, 0);
    if constexpr (GB) stage8_rows(a.rows + t.p0, t.nc, 2);
    if (GATHER) {
      wait_cnt<0>();
      wg_barrier();
    }
    begin_tile(t, 0);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      begin_stage(k, 0);
      load_b(0, k);
      load_a(0, k);
      load_b(1, k);
      load_a(1, k);
      end_stage();
    }
  }
  wait_cnt<12>();   // B half 0 and A half 0 of stage 0 have landed
  wg_barrier();
  read_b(I0{}, I0{});
  wait_cnt<12>();   // every wavefront has read B half 0 of stage 0 before stage 2's replaces it
  wg_barrier();
  if (wm == 1) wg_barrier();   // the second group runs one segment behind the first
  int stores = 0;   // so many stores of the tile before, or more, lie behind the loads in flight: 0 or 16
  for (;; set ^= 1) {
    int nf[2], pairs, rows;
    {
      const Tile t = tiles.tile();
      rows = t.rows;
#pragma unroll
      for (int h = 0; h < 2; ++h) {   // 16-row tiles of each A half that hold rows
        const int v = rows - 128 * h - 16 * wm;
        nf[h] = __builtin_amdgcn_readfirstlane(v >= 128 ? 4 : (v > 0 ? (v + 31) / 32 : 0));
      }
      pairs = (t.nc + 127) / 128;   // pairs of stages: what is not there reads as 0
      if (MODE == kFwd && wave < 2) {   // read behind the loop, 16 loads or more later
        const int64_t j = t.j0 + 128 * wave;
        const u32x4 r = buffer_at(a.bias + t.g * a.bias_group + j, a.bias && a.splits == 1 && j < a.J ? (a.J - j) * 2 : 0);
        load_lds4(r, lane * 4, lds_at(bias_s[set]) + 256 * wave);
      }
    }
    // the tile after this one; after the last its own first stages are loaded again
    const int here = tiles.at;
    const bool last = !tiles.next();
    if (last) tiles.at = here;
    if constexpr (GATHER) {
      const Tile t = tiles.tile();
      if constexpr (GA) tile_rows(a.rows + t.p0, t.rows, set ^ 1);
      if constexpr (GB) stage8_rows(a.rows + t.p0, t.nc, 2 + (set ^ 1));
    }
    if (GB && pairs <= 1) wait_cnt<0>();   // the next tile's row numbers are needed at once

    auto pipeline = [&](auto part) __attribute__((always_inline)) {
      constexpr bool PARTIAL = decltype(part)::value;
      f32x4 acc[2][2][4][2];   // [A half][B half][16-row tile][16-column tile]
#pragma unroll
      for (int ha = 0; ha < 2; ++ha)
#pragma unroll
        for (int hb = 0; hb < 2; ++hb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[ha][hb][i][c] = f32x4{0, 0, 0, 0};
      auto mma = [&](auto ha, auto hb) __attribute__((always_inline)) {
        constexpr int A = decltype(ha)::value, B = decltype(hb)::value;
        auto tile_row = [&](int i, int ks) __attribute__((always_inline)) {
#pragma unroll
          for (int c = 0; c < 2; ++c) acc[A][B][i][c] = T::mma(fw[B][c][ks], ft[i][ks], acc[A][B][i][c]);
        };
        __builtin_amdgcn_s_setprio(1);
        if constexpr (!PARTIAL) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) tile_row(i, ks);
        } else {
#pragma unroll
          for (int i = 0; i < 4; i += 2)
            if (i < nf[A]) {
#pragma unroll
              for (int ks = 0; ks < 2; ++ks) {
                tile_row(i, ks);
                tile_row(i + 1, ks);
              }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        wg_barrier();
      };
      // The next segment's half has landed, this one's fragments are read.  The halves that the first segments wait for
      // were loaded before the stores of the tile before: those may be outstanding too.
      int early = stores ? kTile256Early : 0;
      auto mem_end = [&]() __attribute__((always_inline)) {
        if (early > 0) {
          --early;
          wait_cnt<28>();
        } else {
          wait_cnt<12>();
        }
        wg_barrier();
      };
      // a stage in slot S, loading the stage k of the stream into it
      auto stage = [&](int k, int p, auto ss) __attribute__((always_inline)) {
        constexpr int S = decltype(ss)::value;
        typedef std::integral_constant<int, S> IS;
        typedef std::integral_constant<int, 1 - S> IO;
        begin_stage(k, p);
        read_a(I0{}, IS{});
        load_b(0, S);
        mem_end();
        mma(I0{}, I0{});
        read_b(I1{}, IS{});
        load_a(0, S);
        mem_end();
        mma(I0{}, I1{});
        read_a(I1{}, IS{});
        load_b(1, S);
        mem_end();
        mma(I1{}, I0{});
        read_b(I0{}, IO{});
        load_a(1, S);
        end_stage();
        mem_end();
        mma(I1{}, I1{});
      };
      for (int k = 1; k < pairs; ++k) {
        stage(2 * k, set, I0{});
        stage(2 * k + 1, set, I1{});
      }
      begin_tile(tiles.tile(), set ^ 1);   // the last two stages load the next tile's first two
      stage(0, set ^ 1, I0{});
      stage(1, set ^ 1, I1{});

      const int then = tiles.at;
      tiles.at = here;
      const Tile cur = tiles.tile();
      tiles.at = then;
      const Output<T, MODE, 256, 256> o(a, cur);
      stores = 16;
      int erow = 16 * wm + j16, ecol = 32 * wn + (XB ? 16 * (g4 & 1) + 8 * (g4 >> 1) : 8 * g4);
      asm volatile("" : "+v"(erow), "+v"(ecol));   // the stores' offsets are computed here, not kept through the loop
      const int cols = (int)a.J - cur.j0;
      // a B half's residual is read before its first store: a wait for it behind that would wait for the store too
      auto finish = [&](auto with_res) __attribute__((always_inline)) {
        constexpr bool RES = decltype(with_res)::value;
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
          const int j = ecol + 128 * hb;
          u32x4 res[2][4] = {};
          if constexpr (RES) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 4; ++i) res[h][i] = o.residual(j < cols ? (erow + 128 * h + 32 * i) * o.ldr + j * 2 : kNowhere);
            wait_loads();
          }
          u32x4 bias = {0, 0, 0, 0};
          if constexpr (MODE == kFwd)
            bias = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(bias_s[set]) + j * 2);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              __builtin_amdgcn_sched_barrier(0);   // one row at a time: registers
              const uint32_t r = (uint32_t)(erow + 128 * h + 32 * i);
              float v[8];
              columns8<XB>(acc[h][hb][i][0], acc[h][hb][i][1], v);
              o.template store<ACT>(r * o.ldo, r * o.ldp, j, j < cols, v, bias, res[h][i]);
            }
        }
      };
      if (MODE == kFwd && !GATHER && a.residual && a.splits == 1)
        finish(std::true_type{});
      else
        finish(std::false_type{});
    };
    if (rows >= 256)
      pipeline(std::false_type{});
    else
      pipeline(std::true_type{});
    if (last) break;
  }
  if (wm == 0) wg_barrier();
  wait_cnt<0>();   // no load may write this workgroup's LDS after its end
}

template <typename T, int MODE, bool GATHER, int ACT>
void go(const char* name, const Args& a, int64_t tiles, int64_t cus, hipStream_t s) {
  launch(name, tile256<T, MODE, GATHER, ACT>, dim3((unsigned)std::min(tiles, cus)), dim3(512), 0, s, a);
}

template <typename T>
void tile_typed(int mode, const char* name, const Args& a, int64_t tiles, int64_t cus, hipStream_t s) {
  const bool gather = a.rows != nullptr;
  if (mode == kDx) return go<T, kDx, false, kNone>(name, a, tiles, cus, s);
  if (mode == kDw) return gather ? go<T, kDw, true, kNone>(name, a, tiles, cus, s) : go<T, kDw, false, kNone>(name, a, tiles, cus, s);
  if (gather) return go<T, kFwd, true, kNone>(name, a, tiles, cus, s);
  switch (a.splits > 1 ? kNone : a.act) {
    case kRelu: return go<T, kFwd, false, kRelu>(name, a, tiles, cus, s);
    case kSilu: return go<T, kFwd, false, kSilu>(name, a, tiles, cus, s);
    case kGelu: return go<T, kFwd, false, kGelu>(name, a, tiles, cus, s);
    case kGeluTanh: return go<T, kFwd, false, kGeluTanh>(name, a, tiles, cus, s);
    default: return go<T, kFwd, false, kNone>(name, a, tiles, cus, s);
  }
}

}  // namespace

void tile_launch(int mode, int32_t dtype, const char* name, const Args& a, int64_t tiles, int64_t cus, hipStream_t s) {
  dtype == FERRY_BF16 ? tile_typed<Bf16>(mode, name, a, tiles, cus, s) : tile_typed<F16>(mode, name, a, tiles, cus, s);
}

}  // namespace lin
}  // namespace ferry
