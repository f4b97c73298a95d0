// Launches of the linear products' tiled kernels (linear_tile.hip).
#pragma once

#include "linear.h"

namespace ferry {
namespace lin {

// 256 x 256 tiles, `tiles` of them at most, on `cus` CUs
void tile_launch(int mode, int32_t dtype, const char* name, const Args& a, int64_t tiles, int64_t cus, hipStream_t s);

}  // namespace lin
}  // namespace ferry
