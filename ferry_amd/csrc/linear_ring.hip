// The linear products on tiles smaller than 256 x 256: where few rows, columns or tiles leave CUs idle with those.
#include "linear_plan.h"
#include "linear_stream.h"
#include "linear_tile.h"

#include <algorithm>
#include <climits>

namespace ferry {
namespace lin {
namespace {

// TM = 16 WM MI indices of A by TN = 16 WN NI of B per workgroup of WM x WN wavefronts, each with MI x NI
// accumulators of 16 x 16.  Stages of 64 of the contraction stream through an LDS ring as deep as 144 KiB allows
// (3 to 9; 128 KiB beside row numbers), one barrier a stage; the loads of a stage are issued between the products of another.  The stream
// of loads runs ahead of the products by the whole ring, over the ends of tiles, however short these are: it
// keeps its own place in the list of tiles, and loads nothing (zeros) behind the last one, so that a stage is
// always the same number of loads and one constant says that the next stage has landed.  Bound by reading the
// operands where rows are few, by latency and LDS reads elsewhere.
template <typename T, int MODE, bool GATHER, int WM, int WN, int MI, int NI>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(WM * WN / 4, WM * WN / 4))) void ring_kernel(Args a) {
  constexpr bool XA = MODE == kDw, XB = MODE != kFwd, RAG = MODE != kDw;
  constexpr bool GA = GATHER && MODE == kFwd, GB = GATHER && MODE == kDw;
  constexpr int W = WM * WN, TM = 16 * WM * MI, TN = 16 * WN * NI;
  constexpr int kStage = (TM + TN) * 128, SST = ring_stages(TM, TN, GB);
  constexpr int LA = TM / (8 * W), LB = TN / (8 * W), LPS = LA + LB;   // loads of a wavefront and stage
  // GB: rows of x of a wavefront and stage, stages whose row numbers 64 lanes load at once
  constexpr int RPW = LB * 512 / TN, BS = 64 / RPW;
  __shared__ Table tt;
  __shared__ typename Tiles<MODE, GATHER, TM, TN>::Store places;
  __shared__ __attribute__((aligned(1024))) char smem[SST * kStage];
  // row numbers (low and high words), each wavefront its own.  GA: of a tile, two in turn.  GB: of BS stages,
  // sets 0 and 1 in turn, 2 and 3 for the first ones of a tile.
  __shared__ __attribute__((aligned(256))) uint32_t row_s[GA ? 2 : (GB ? 4 : 1)][2][GATHER ? 64 * W : 1];
  __shared__ __attribute__((aligned(256))) uint32_t bias_s[MODE == kFwd ? 2 : 1][MODE == kFwd ? 64 : 1];   // as in tile256
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  build_table<RAG>(a, tt, RAG ? TM : (int)ceil_div(a.I, TM));
  if (RAG && a.zero_rest) zero_rest(a, tt.first, tt.last);
  Tiles<MODE, GATHER, TM, TN> tiles(a, tt, places);   // of the products
  if (!tiles.next()) return;
  Tiles<MODE, GATHER, TM, TN> ahead = tiles;          // of the stream of loads
  const int wm = wave / WN, wn = wave % WN;
  const int j16 = lane & 15, g4 = lane >> 4;
  const uint32_t smem0 = lds_at(smem);
  const uint32_t lda2 = (uint32_t)a.lda * 2, ldb2 = (uint32_t)a.ldb * 2;
  const uint32_t a_step = XA ? 64 * lda2 : 128, b_step = XB ? (GB ? 0 : 64 * ldb2) : 128;

  // fragment reads: tile i of A 16 WM i + 16 wm + [0, 16), of B 16 NI wn + 16 c (staged by index: pairs interleaved)
  uint32_t a_addr[XA ? MI : 2], b_addr[XB ? NI : 2];
  if constexpr (XA) {
#pragma unroll
    for (int i = 0; i < MI; ++i) a_addr[i] = smem0 + frag_across<TM>(16 * WM * i + 16 * wm, 0, 0);
  } else {
    const int r = 16 * wm + j16;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) a_addr[ks] = smem0 + (uint32_t)(r * 128 + (((4 * ks + g4) ^ swz_direct(r)) << 4));
  }
  if constexpr (XB) {
#pragma unroll
    for (int c = 0; c < NI; ++c) b_addr[c] = smem0 + TM * 128 + frag_across<TN>(16 * NI * wn + 16 * c, 0, 0);
  } else {
    const int r = 16 * NI * wn + 8 * (j16 >> 2) + (j16 & 3);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) b_addr[ks] = smem0 + TM * 128 + (uint32_t)(r * 128 + (((4 * ks + g4) ^ swz_pair(r)) << 4));
  }

  // -- the stream of loads --
  u32x4 ra, rb;
  uint32_t sa = 0, sb = 0, avo[LA], bvo[LB];
  int left = 0, sk = 0, skt = 0, set = 0;   // set: GA the tile's, GB 2 + set its first
  const int64_t* idx = nullptr;
  // row r of the wavefront's load q of an operand, and the chunk of the row that the lane loads
  auto row_a = [&](int q) __attribute__((always_inline)) {
    return XA ? 512 / TM * (LA * wave + q) + lane / (TM / 8) : 8 * (LA * wave + q) + (lane >> 3);
  };
  auto row_b = [&](int q) __attribute__((always_inline)) {
    return XB ? 512 / TN * (LB * wave + q) + lane / (TN / 8) : 8 * (LB * wave + q) + (lane >> 3);
  };
  auto chunk_a = [&](int q) __attribute__((always_inline)) {
    return XA ? (lane % (TM / 8)) ^ swz_across<TM>(row_a(q)) : (lane & 7) ^ swz_direct(row_a(q));
  };
  auto chunk_b = [&](int q) __attribute__((always_inline)) {
    return XB ? (lane % (TN / 8)) ^ swz_across<TN>(row_b(q)) : (lane & 7) ^ swz_pair(row_b(q));
  };
  auto tile_rows = [&](const Tile& t, int p) __attribute__((always_inline)) {   // GA: of the wavefront's rows
    const u32x4 r = buffer_at(a.rows + t.p0, (int64_t)(t.rows < TM ? t.rows : TM) * 8);
    const uint32_t o = lane < 8 * LA ? (uint32_t)(8 * LA * wave + lane) * 8 : kNowhere;
    load_lds4(r, o, lds_at(row_s[p][0]) + 256 * wave);
    load_lds4(r, o == kNowhere ? o : o + 4, lds_at(row_s[p][1]) + 256 * wave);
  };
  auto stage_rows = [&](const int64_t* at, int n, int p) __attribute__((always_inline)) {   // GB: of the wavefront's rows of BS stages
    const u32x4 r = buffer_at(at, (int64_t)n * 8);
    const uint32_t o = (uint32_t)(lane / RPW * 64 + RPW * wave + lane % RPW) * 8;
    load_lds4(r, o, lds_at(row_s[p][0]) + 256 * wave);
    load_lds4(r, o + 4, lds_at(row_s[p][1]) + 256 * wave);
  };
  auto begin_tile = [&](const Tile& t) __attribute__((always_inline)) {
    ra = t.a, rb = t.b, sa = sb = 0, left = t.nc, sk = 0;
    if constexpr (GB) idx = a.rows + t.p0;
    skt = t.nc > 64 ? (t.nc + 63) / 64 : 1;
#pragma unroll
    for (int q = 0; q < LA; ++q) {
      if constexpr (GA) {
        const uint32_t x = row_s[set][0][64 * wave + 8 * q + (lane >> 3)];
        const bool ok = row_a(q) < t.rows && row_s[set][1][64 * wave + 8 * q + (lane >> 3)] == 0 && x < (uint64_t)a.x_rows;
        avo[q] = ok ? x * lda2 + chunk_a(q) * 16 : kNowhere;
      } else {
        avo[q] = (uint32_t)row_a(q) * lda2 + chunk_a(q) * 16;
      }
    }
    if constexpr (!GB) {
#pragma unroll
      for (int q = 0; q < LB; ++q) bvo[q] = (uint32_t)row_b(q) * ldb2 + chunk_b(q) * 16;
    }
    if constexpr (GATHER) {   // the row numbers of the tile after this one
      Tiles<MODE, GATHER, TM, TN> next = ahead;
      const Tile n = next.next() ? next.tile() : t;
      if constexpr (GA) tile_rows(n, set ^ 1);
      if constexpr (GB) stage_rows(a.rows + n.p0, n.nc, 2 + (set ^ 1));
    }
  };
  auto begin_stage = [&]() __attribute__((always_inline)) {   // before a stage is loaded
    if (left <= 0) {   // not there: zeros
      ra[2] = rb[2] = 0;
      sa = sb = 0;
    } else if (!(XA && XB) && left < 64) {   // chunks behind the contraction's end lie nowhere
#pragma unroll
      for (int q = 0; q < LA; ++q)
        if constexpr (!XA) avo[q] = chunk_a(q) * 8 >= left ? kNowhere : avo[q];
#pragma unroll
      for (int q = 0; q < LB; ++q)
        if constexpr (!XB) bvo[q] = chunk_b(q) * 8 >= left ? kNowhere : bvo[q];
    }
    if constexpr (GB) {
      if (sk % BS == 0) {
        // this batch was loaded BS stages ago: landed, unless the ring is deeper than that
        if (BS < SST && sk) wait_cnt<BS * LPS>();
        if (left > 64 * BS) stage_rows(idx + 64 * BS, left - 64 * BS, (sk / BS + 1) & 1);
        idx += 64 * BS;
      }
      const int p = sk < BS ? 2 + set : (sk / BS) & 1;
#pragma unroll
      for (int q = 0; q < LB; ++q) {
        const int r = row_b(q), at = 64 * wave + RPW * (sk % BS) + r - RPW * wave;
        const uint32_t x = row_s[p][0][at];
        const bool ok = r < left && row_s[p][1][at] == 0 && x < (uint64_t)a.x_rows;
        bvo[q] = ok ? x * ldb2 + chunk_b(q) * 16 : kNowhere;
      }
    }
  };
  auto load = [&](auto qq, int slot) __attribute__((always_inline)) {
    constexpr int q = decltype(qq)::value;
    const uint32_t dst = smem0 + (uint32_t)(slot * kStage);
    if constexpr (q < LA)
      load_lds(ra, avo[q], sa, dst + 1024 * (LA * wave + q));
    else
      load_lds(rb, bvo[q - LA], sb, dst + TM * 128 + 1024 * (LB * wave + q - LA));
  };
  auto end_stage = [&](bool filling) __attribute__((always_inline)) {
    left -= 64;
    sa += a_step;
    sb += b_step;
    if (++sk < skt) return;
    const int kt = skt;
    if (ahead.next()) {
      if (GATHER && ring_rows_wait(kt, SST, filling)) wait_cnt<0>();   // its row numbers were loaded kt stages ago
      set ^= 1;
      begin_tile(ahead.tile());
    } else {
      left = 0;
      sk = 1;
      skt = INT_MAX;
    }
  };

  s16x8 t0[MI], w0[NI], t1[MI], w1[NI];
  auto read = [&](int slot, auto kk, s16x8 (&ft)[MI], s16x8 (&fw)[NI]) __attribute__((always_inline)) {
    constexpr int KS = decltype(kk)::value;
    const uint32_t st = slot * kStage;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      if constexpr (XB)
        fw[c] = read_across(b_addr[c] + st + KS * 64 * TN, b_addr[c] + st + KS * 64 * TN + 8 * TN);
      else
        fw[c] = read_direct(b_addr[KS] + st + (c >> 1) * 32 * 128 + (c & 1) * 4 * 128);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      if constexpr (XA)
        ft[i] = read_across(a_addr[i] + st + KS * 64 * TM, a_addr[i] + st + KS * 64 * TM + 8 * TM);
      else
        ft[i] = read_direct(a_addr[KS] + st + i * 16 * WM * 128);
    }
  };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;

  {
    const Tile t = tiles.tile();
    if constexpr (GA) tile_rows(t, 0);
    if constexpr (GB) stage_rows(a.rows + t.p0, t.nc, 2);
    if (GATHER) wait_cnt<0>();
    begin_tile(t);
  }
  for (int k = 0; k < SST; ++k) {
    begin_stage();
    static_for<0, LPS>([&](auto q) __attribute__((always_inline)) { load(q, k); });
    end_stage(true);
  }
  wait_cnt<(SST - 1) * LPS>();
  wg_barrier();
  read(0, I0{}, t0, w0);
  int cur = 0;   // slot of the stage
  constexpr int kStores = MI * NI / 2;   // of a wavefront and whole tile
  int early = 0;   // stages whose loads are older than the stores of the tile before
  int bs = 0;
  for (bool more = true; more; more = tiles.next(), bs ^= 1) {
    const Tile t = tiles.tile();
    const int kt = t.nc > 64 ? (t.nc + 63) / 64 : 1;
    const int v = t.rows - 16 * wm;   // 16-row tiles of this wavefront that hold rows
    const int nf = __builtin_amdgcn_readfirstlane(v <= 0 ? 0 : ((v + 16 * WM - 1) / (16 * WM) < MI ? (v + 16 * WM - 1) / (16 * WM) : MI));
    if (MODE == kFwd && wave == 0) {   // (128 columns)
      const u32x4 r = buffer_at(a.bias + t.g * a.bias_group + t.j0, a.bias && a.splits == 1 ? (a.J - t.j0) * 2 : 0);
      load_lds4(r, lane * 4, lds_at(bias_s[bs]));
    }
    f32x4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int c = 0; c < NI; ++c) acc[i][c] = f32x4{0, 0, 0, 0};
    auto mma = [&](int i, const s16x8 (&ft)[MI], const s16x8 (&fw)[NI]) __attribute__((always_inline)) {
      if (i < nf) {
#pragma unroll
        for (int c = 0; c < NI; ++c) acc[i][c] = T::mma(fw[c], ft[i], acc[i][c]);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int k = 0; k < kt; ++k) {
      const int nxt = cur + 1 == SST ? 0 : cur + 1;
      read(cur, I1{}, t1, w1);
#pragma unroll
      for (int i = 0; i < MI; ++i) mma(i, t0, w0);
      // the stage is read by this wavefront, its loads of the next have landed
      if (early > 0) {   // the stores of the tile before may be outstanding too
        --early;
        wait_cnt<(SST - 2) * LPS + kStores>();
      } else {
        wait_cnt<(SST - 2) * LPS>();
      }
      wg_barrier();
      read(nxt, I0{}, t0, w0);
      begin_stage();
      static_for<0, MI>([&](auto ii) __attribute__((always_inline)) {
        constexpr int i = decltype(ii)::value;
        static_for<i * LPS / MI, (i + 1) * LPS / MI>([&](auto q) __attribute__((always_inline)) { load(q, cur); });
        mma(i, t1, w1);
      });
      end_stage(false);
      cur = nxt;
    }
    if (MODE == kFwd && kt < SST) {   // the bias was loaded at the tile's start
      wait_cnt<0>();
      wg_barrier();
    }
    const Output<T, MODE, TM, TN> o(a, t);
    early = SST - 1;
    const int cols = (int)a.J - t.j0, ecol = 16 * NI * wn + (XB ? 16 * (g4 & 1) + 8 * (g4 >> 1) : 8 * g4);
    // the residual is read before the first store, as in tile256
    auto finish = [&](auto with_res) __attribute__((always_inline)) {
      constexpr bool RES = decltype(with_res)::value;
      u32x4 res[NI / 2][MI] = {};
      if constexpr (RES) {
#pragma unroll
        for (int cc = 0; cc < NI / 2; ++cc)
#pragma unroll
          for (int i = 0; i < MI; ++i)
            res[cc][i] = o.residual(ecol + 32 * cc < cols ? (16 * WM * i + 16 * wm + j16) * o.ldr + (ecol + 32 * cc) * 2 : kNowhere);
        wait_loads();
      }
#pragma unroll
      for (int cc = 0; cc < NI / 2; ++cc) {
        const int j = ecol + 32 * cc;
        u32x4 bias = {0, 0, 0, 0};
        if constexpr (MODE == kFwd)
          bias = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(bias_s[bs]) + j * 2);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const uint32_t r = (uint32_t)(16 * WM * i + 16 * wm + j16);
          float v8[8];
          columns8<XB>(acc[i][2 * cc], acc[i][2 * cc + 1], v8);
          o.template store<MODE == kFwd && !GATHER ? -1 : (int)kNone>(r * o.ldo, r * o.ldp, j, j < cols, v8, bias, res[cc][i]);
        }
      }
    };
    if (MODE == kFwd && !GATHER && a.residual && a.splits == 1)
      finish(std::true_type{});
    else
      finish(std::false_type{});
  }
  wait_cnt<0>();   // no load may write this workgroup's LDS after its end
}

template <typename T, int MODE, bool GATHER>
void ring_shape(int shape, const char* name, const Args& a, int64_t tiles, int64_t cus, hipStream_t s) {
  auto go = [&](auto kernel, int threads) {
    launch(name, kernel, dim3((unsigned)std::min(tiles, cus)), dim3(threads), 0, s, a);
  };
  switch (shape) {
    case 1:   // (no third stage beside the row numbers of a gathered x)
      if constexpr (!(GATHER && MODE == kDw)) return go(ring_kernel<T, MODE, GATHER, 4, 2, 4, 4>, 512);
      [[fallthrough]];
    case 2: return go(ring_kernel<T, MODE, GATHER, 4, 2, 2, 4>, 512);
    case 3: return go(ring_kernel<T, MODE, GATHER, 2, 4, 2, 2>, 512);
    default: return go(ring_kernel<T, MODE, GATHER, 2, 2, 2, 2>, 256);
  }
}
template <typename T>
void ring_typed(int mode, int shape, const char* name, const Args& a, int64_t tiles, int64_t cus, hipStream_t s) {
  const bool gather = a.rows != nullptr;
  if (mode == kDx) return ring_shape<T, kDx, false>(shape, name, a, tiles, cus, s);
  if (mode == kDw) return gather ? ring_shape<T, kDw, true>(shape, name, a, tiles, cus, s) : ring_shape<T, kDw, false>(shape, name, a, tiles, cus, s);
  return gather ? ring_shape<T, kFwd, true>(shape, name, a, tiles, cus, s) : ring_shape<T, kFwd, false>(shape, name, a, tiles, cus, s);
}

}  // namespace

void ring_launch(int mode, int32_t dtype, int shape, const char* name, const Args& a, int64_t tiles, int64_t cus, hipStream_t s) {
  dtype == FERRY_BF16 ? ring_typed<Bf16>(mode, shape, name, a, tiles, cus, s) : ring_typed<F16>(mode, shape, name, a, tiles, cus, s);
}

}  // namespace lin
}  // namespace ferry
