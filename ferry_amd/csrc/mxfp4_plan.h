// How the launches of the MXFP4 expert FFN with tiles are cut: host arithmetic only.
#pragma once

#include <cstdint>

namespace ferry {

struct MxPlan {
  bool large;        // 4-bit activations: tiles of 256 x 256, one workgroup on a CU; otherwise two
  int tile_rows;
  int tile_wgs;      // workgroups that take tiles, one after the other
  int items;         // small experts: groups of weight rows of a workgroup
  int small_wgs;     // small experts' workgroups behind the tiles; 0 with spare CUs: a launch of their own
};

// Items of a workgroup of small experts, a power of two that divides an expert's (cols), so many that at most `per_cu`
// workgroups come to a CU: those that run at once by their LDS (up at 16 tokens 13.5 us, with one item a workgroup 17.5,
// with 4-bit activations 12 and 15.5), behind tiles twice as many, which level the end (256 tokens of 64 experts of 2048
// x 1408 53 + 35 us, with half as many 58 + 40, with one item each 64 + 35).
inline int small_items(int experts, int cols, int64_t per_cu, int64_t cus) {
  int items = 1;
  while (cols % (2 * items) == 0 && (int64_t)experts * (cols / items) > per_cu * cus) items *= 2;
  return items;
}

// One projection.  col_tiles: tiles of 256 weight rows; tiles: the row tiles of 256, 128 and 64 rows of the larger experts
// (upper bounds); small, small_cols: the small experts and an expert's items.
//
// 4-bit activations: the large tiles where the rows make at least six quarters of them for each CU.  Up and down, large
// tiles against small ones: 512 tokens (128 experts of 2048 x 768, top 8, Zipf 1.1; 1.2 and 1.6 quarters) 43 + 32 us
// against 39 + 29, 2,048 tokens (7 and 9.4) 78 + 54 against 79 + 54, 4,096 (13 and 17) 113 + 79 against 120
// + 84; evenly spread, 1,024 tokens (3 and 4) 62 + 37 against 56 + 36, 2,048 (6 and 8) 72 + 46 against 79 + 52.
// Tiles of 128 rows become tiles of 64 where each has a CU of its own: they read the weights twice, and the longest
// takes less time.  Up and down, bf16 activations (128 experts of 2048 x 768, top 8, Zipf 1.1): 100 tokens 34 + 19
// us against 28 + 18; 64 rows two to a CU, and 32, were level with these or slower (29 + 19).
//
// The small experts' workgroups come behind those of the tiles and run where a CU has no tile (left): up + down, with
// bf16 and with 4-bit activations, 20 tokens took 37 and 37 us, with launches of their own 57 and 49, 777 tokens (64
// experts of 2048 x 1408, top 6) 13 and 10 % less than with these, 8,192 tokens 2 and 6 %; before the tiles' they
// delay them (777 tokens 12 and 6 % more than behind).
//
// spare: the tiles' launch leaves the room of that many CUs to other streams' kernels (at least 8 are used).  Nothing
// comes behind the tiles then, so that what is left is not filled; where two of its workgroups share a CU, the room may be
// half of twice as many CUs.
inline MxPlan plan_tiles(bool quantised, int64_t col_tiles, const int64_t (&tiles)[3], int small, int small_cols, int64_t cus,
                         int64_t spare) {
  MxPlan p;
  if (spare > 0) cus = cus - spare > 8 ? cus - spare : 8;
  p.large = quantised && tiles[2] * col_tiles >= 6 * cus;
  const int64_t cols = quantised && !p.large ? 2 * col_tiles : col_tiles, most = (p.large ? cus : 2 * cus) / 8 * 8;
  const int by = p.large ? 0 : tiles[2] * cols <= cus ? 2 : 1;
  p.tile_rows = 256 >> by;
  const int64_t t = tiles[by] * cols;
  p.tile_wgs = (int)(t < most ? (t + 7) / 8 * 8 : most);
  const int items = small_cols / (p.large ? 2 : 1);   // a workgroup of the large tiles does two workgroups' work
  p.items = small_items(small, items, p.large ? 2 : 4, cus);
  p.small_wgs = spare > 0 ? 0 : small * (items / p.items);
  return p;
}

}  // namespace ferry
