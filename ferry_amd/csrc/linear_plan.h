// Arithmetic of the linear products' launches and pipelines that needs no device: also built by itself, for tests.
#pragma once

#include <cstdint>

namespace ferry {
namespace lin {

// ring_kernel's stages of 64 of the contraction: as many as 144 KiB hold, 128 KiB beside the row numbers of a gathered dW
constexpr int ring_stages(int tm, int tn, bool gathered_dw) { return (gathered_dw ? 131072 : 147456) / ((tm + tn) * 128); }

// Whether ring_kernel's loads are awaited where the stream goes on behind a tile of kt stages: the next tile's row
// numbers were loaded where this one began.  In the loop each stage waits until the loads of ring - 2 stages at most are
// outstanding, so kt >= ring - 1 stages suffice; the stages that fill the ring wait for nothing.
constexpr bool ring_rows_wait(int kt, int ring, bool filling) { return kt < ring + (filling ? 1 : 0); }

// tile256's phases behind the stores of the tile before in which these may be outstanding as well.  The phase's wait is for
// the half that the next phase reads.  Eight halves were loaded before the stores; the first was awaited there, the
// second too, with the products' last phase, and the other six are awaited by the first six phases.  What the seventh
// awaits was loaded behind the stores.
constexpr int kTile256Early = 6;

// A contraction of c in parts: each but the last has part_length, the last what is left, which may be little or nothing.
constexpr int64_t part_length(int64_t c, int64_t parts) { return ((c + parts - 1) / parts + 63) / 64 * 64; }
constexpr int64_t last_part(int64_t c, int64_t parts) {
  return c > (parts - 1) * part_length(c, parts) ? c - (parts - 1) * part_length(c, parts) : 0;
}

// Whether tile256 takes a gathered x whose contraction is cut into these parts: it loads the row numbers of a tile where the
// tile before begins and awaits them with that tile's stages, all but the last two, so every part needs more than two.
constexpr bool tile256_gathers(int64_t c, int64_t parts) { return last_part(c, parts) > 128; }

// Bytes from tile256's first half of an operand (128 indices) to its second, for an operand of `there` indices from the tile's
// first on, staged across (by the contraction) or directly (by rows of ld2 bytes).  A second half without indices loads
// the first again: its offset would lie behind the end of a buffer whose last row is short, where the hardware's
// comparison with size - offset wraps and keeps no lane inside.
constexpr uint32_t half_offset(bool across, int64_t there, uint32_t ld2) { return there > 128 ? (across ? 256 : 128 * ld2) : 0; }

}  // namespace lin
}  // namespace ferry
