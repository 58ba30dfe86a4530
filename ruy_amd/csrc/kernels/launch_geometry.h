// Launch geometry of the kernels whose grids follow the problem size in more
// than one dimension. Plain host arithmetic, kept apart from the kernels so
// that its bounds can be tested without a device.
#ifndef RUY_AMD_CSRC_KERNELS_LAUNCH_GEOMETRY_H_
#define RUY_AMD_CSRC_KERNELS_LAUNCH_GEOMETRY_H_

#include <cstdint>

namespace ruyamd {

// HIP limits: grid.x < 2^31, grid.y and grid.z <= 65535, fewer than 2^32 threads along a dimension.
constexpr unsigned kMaxGridX = 0x7fffffffu;
constexpr unsigned kMaxGridY = 65535u;

// Whether `blocks` workgroups of `threads` can be launched along x.
inline bool LaunchFits(int64_t blocks, int threads) {
  return blocks <= int64_t(kMaxGridX) && blocks * threads <= int64_t(0xffffffff);
}

struct Grid2D {
  unsigned x = 1;
  unsigned y = 1;
};

// Generic kernel: tiles of kGenericTile x kGenericTile destination elements,
// x along the destination's contiguous dimension (`fast` elements), y along
// the other (`slow` elements). The kernel walks tile rows blockIdx.y,
// blockIdx.y + gridDim.y, ... so y may be capped.
constexpr int kGenericTile = 16;
inline Grid2D GenericGrid(int fast, int slow) {
  Grid2D g;
  const int64_t bx = (int64_t(fast) + kGenericTile - 1) / kGenericTile;
  const int64_t by = (int64_t(slow) + kGenericTile - 1) / kGenericTile;
  g.x = static_cast<unsigned>(bx < 1 ? 1 : bx);  // at most 2^27 for an int dimension
  g.y = static_cast<unsigned>(by < 1 ? 1 : (by > int64_t(kMaxGridY) ? int64_t(kMaxGridY) : by));
  return g;
}

// Element-wise kernels: `threads` elements per workgroup, grid-stride loop, so
// the block count may be capped as well.
inline unsigned ElementwiseBlocks(int64_t n, int threads) {
  const int64_t b = (n + threads - 1) / threads;
  return static_cast<unsigned>(b < 1 ? 1 : (b > int64_t(kMaxGridX) ? int64_t(kMaxGridX) : b));
}

// Whether what a tile reads of `runs` runs, `pitch` bytes from one to the next and the first `length` bytes of each,
// ends within the 2^31 bytes that a buffer resource of the tiled grouped kernel has. (What lies beyond
// its end is read as zeros, with no error.)
inline bool TileOffsetsFit(int64_t runs, int64_t pitch, int64_t length) {
  return (runs - 1) * pitch + length <= int64_t(1) << 31;
}

// Tiles dealt to the eight XCDs, each of which makes so many at once (where it has no CU of its own, one): what is left of an XCD's
// share after full rounds of these goes to four workgroups a tile where it is a quarter of a round at most. The host's
// count of workgroups and the device's search go by these, whatever the number of CUs.
constexpr int TilesAtOnce(int compute_units) { return compute_units < 8 ? 1 : compute_units / 8; }

// What workgroup number `place` of an XCD that has `tiles` tiles makes: tile number `tile` of these (`tiles` and more: none), or
// one quarter of it (-1: all of it).
struct XcdPlace {
  int64_t tile;
  int quarter;
};
constexpr XcdPlace XcdPlaceOf(int64_t place, int64_t tiles, int at_once) {
  const int64_t full = tiles / at_once * at_once;
  if (!full || place < full || (tiles - full) * 4 > at_once) return {place, -1};
  return {full + (place - full) / 4, static_cast<int>((place - full) & 3)};
}

// Workgroups that an XCD with `tiles` tiles (or_fewer: or any number below) needs at most.
constexpr int64_t XcdWorkgroups(int64_t tiles, int at_once, bool or_fewer) {
  if (tiles < at_once) return tiles;
  const int64_t rest = tiles % at_once;
  return tiles + 3 * (or_fewer ? at_once / 4 : rest * 4 <= at_once ? rest : 0);
}

}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_LAUNCH_GEOMETRY_H_
