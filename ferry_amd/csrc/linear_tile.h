// Launches of the linear products' kernels for aligned operands (linear_tile.hip,
// linear_ring.hip, linear_few.hip).
#pragma once

#include "linear.h"

namespace ferry {
namespace lin {

// 256 x 256 tiles, `tiles` of them at most, on `cus` CUs
void tile_launch(int mode, int32_t dtype, const char* name, const Args& a, int64_t tiles, int64_t cus, hipStream_t s);

// smaller tiles, shape 1 to 4: 256 x 128, 128 x 128, 64 x 128, 64 x 64 (indices of A by those of B)
void ring_launch(int mode, int32_t dtype, int shape, const char* name, const Args& a, int64_t tiles, int64_t cus, hipStream_t s);
// kFwd and kDx of few rows: tiles of 16 mt rows, at most `tiles` of them, by 16 nb columns
void few_launch(int mode, int32_t dtype, int mt, int nb, const Args& a, int64_t tiles, int64_t cus, hipStream_t s);

}  // namespace lin
}  // namespace ferry
