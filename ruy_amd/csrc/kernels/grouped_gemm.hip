// Launches of the tiled kernel of grouped products.
#include "grouped_gemm.h"
#include "launch_geometry.h"

#include <algorithm>
#include <cmath>
#include <iterator>

namespace ruyamd {
namespace grouped {
namespace {

enum class Tile { k64x64, k128x128, k256x128, k256x256 };

struct Grid {
  unsigned blocks;
  Tile tile;
  bool far;  // kFar of the kernel
};

// A tile's sizes, the threads of its workgroup, the workgroups that a CU runs side by side, and how long one step
// of all of them takes, with operands straight to LDS, through registers, and fp32 (0: there is no such
// kernel). Measured on each tile in that order, us: bfloat16, 8 x 4096 x 2048 x 8192
// 265 / 181 / 167 / 171, 16 x 1683 x 3968 x 6400 194 / 147 / 133 / 116; through registers, 4 x 4095 x 2047 x 8191
// 367 / 239 / 207, 16 x 1001 x 501 x 2001 10.8 / 18.2 / 19.2 (128x128 is nowhere the best there and left out).
struct TileCost {
  Tile tile;
  int m, n, threads, per_cu;
  float direct, through, f32;
};
constexpr TileCost kTiles[] = {{Tile::k64x64, 64, 64, 256, 2, 0.48f, 0.58f, 1.05f},
                               {Tile::k128x128, 128, 128, 256, 2, 1.08f, 0, 3.9f},
                               {Tile::k256x128, 256, 128, 512, 1, 1.0f, 1.6f, 0},
                               {Tile::k256x256, 256, 256, 512, 1, 1.68f, 0, 0}};
// What a workgroup does before its first step and after its last, in steps.
constexpr float kFixedSteps = 6;

template <int kType, Runs kRunsM, Runs kRunsN, int kWavesM, int kWavesN, int kBlocksM, int kBlocksN, bool kDirect, int kStages,
          bool kFar = false>
void LaunchKernel(hipStream_t stream, const GemmArgs& args, unsigned blocks) {
  constexpr int kLds = kStages * (kWavesM * kBlocksM + kWavesN * kBlocksN) * 16 * 128;
  auto* const kernel = &GroupedGemmKernel<kType, kRunsM, kRunsN, kWavesM, kWavesN, kBlocksM, kBlocksN, kDirect, kStages, kFar>;
  static const hipError_t attribute = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  (void)attribute;  // (a launch that needs it fails)
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWavesM * kWavesN), kLds, stream, args);
}

// (Eight waves on the larger tiles, four on the others.)
template <int kType, Runs kRunsM, Runs kRunsN, bool kDirect>
void LaunchOne(hipStream_t stream, const GemmArgs& args, const Grid& grid) {
  if constexpr (kType != RUYAMD_DTYPE_F32) {
    if constexpr (kDirect)
      if (grid.tile == Tile::k256x256)
        return LaunchKernel<kType, kRunsM, kRunsN, 2, 4, 8, 4, true, 2>(stream, args, grid.blocks);
    if (grid.tile == Tile::k256x128)
      return LaunchKernel<kType, kRunsM, kRunsN, 4, 2, 4, 4, kDirect, kDirect ? 3 : 2>(stream, args, grid.blocks);
  }
  if constexpr (kDirect)
    if (grid.tile == Tile::k128x128)
      return LaunchKernel<kType, kRunsM, kRunsN, 2, 2, 4, 4, true, 2>(stream, args, grid.blocks);
  if constexpr (!kDirect && (kRunsM == Runs::kPlain || kRunsN == Runs::kPlain))
    if (grid.far) return LaunchKernel<kType, kRunsM, kRunsN, 2, 2, 2, 2, false, 2, true>(stream, args, grid.blocks);
  LaunchKernel<kType, kRunsM, kRunsN, 2, 2, 2, 2, kDirect, kDirect ? 4 : 2>(stream, args, grid.blocks);
}

template <int kType, bool kDirect>
void LaunchRuns(hipStream_t stream, const GemmArgs& args, Runs m, Runs n, const Grid& grid) {
  if (m == Runs::kPlain && n == Runs::kPlain) return LaunchOne<kType, Runs::kPlain, Runs::kPlain, kDirect>(stream, args, grid);
  if (m == Runs::kPlain) return LaunchOne<kType, Runs::kPlain, Runs::kAcross, kDirect>(stream, args, grid);
  if (n == Runs::kPlain) return LaunchOne<kType, Runs::kAcross, Runs::kPlain, kDirect>(stream, args, grid);
  LaunchOne<kType, Runs::kAcross, Runs::kAcross, kDirect>(stream, args, grid);
}

template <bool kDirect>
void LaunchType(hipStream_t stream, const GemmArgs& args, int type, Runs m, Runs n, const Grid& grid) {
  if (type == RUYAMD_DTYPE_BF16) return LaunchRuns<RUYAMD_DTYPE_BF16, kDirect>(stream, args, m, n, grid);
  if (type == RUYAMD_DTYPE_F16) return LaunchRuns<RUYAMD_DTYPE_F16, kDirect>(stream, args, m, n, grid);
  LaunchRuns<RUYAMD_DTYPE_F32, kDirect>(stream, args, m, n, grid);
}

}  // namespace

bool LaunchTiles(hipStream_t stream, const Call& call, hipError_t* status) {
  const int bytes = call.type == RUYAMD_DTYPE_F32 ? 4 : 2, granule = 16 / bytes;
  const bool columns = call.dealt == Dealt::kColumns;
  // The M side is the one along which dst is contiguous. (Columns that are dealt
  // to groups stay on the N side; a dst by rows is then written value by value.)
  const bool swapped = !columns && call.dst_rs != 1;
  GemmArgs a;
  a.dealt = call.dealt;
  a.depth = call.k;
  a.offsets = call.offsets;
  a.groups = call.groups;
  a.bias = call.bias;
  a.bias_stride = call.bias_stride;
  a.clamp_min = call.clamp_min;
  a.clamp_max = call.clamp_max;
  a.dst = call.dst;
  a.dst_f32 = call.dst_type == RUYAMD_DTYPE_F32;
  a.dst_group_stride = columns ? 0 : call.matrix_stride;
  const auto side = [&](bool lhs, Side* s) {
    const int64_t along = lhs ? call.lhs_rs : call.rhs_cs, depth = lhs ? call.lhs_cs : call.rhs_rs;
    s->data = lhs ? call.lhs : call.rhs;
    s->count = lhs ? call.m : call.n;
    s->group_stride = columns && lhs ? call.matrix_stride : 0;
    // (A side of one row, or a depth of one, has both strides 1: either order will do.)
    const Runs runs = depth == 1 ? Runs::kPlain : Runs::kAcross;
    s->pitch = runs == Runs::kPlain ? along : depth;
    return runs;
  };
  const Runs runs_m = side(!swapped, &a.m), runs_n = side(swapped, &a.n);
  a.dst_m_stride = swapped ? call.dst_cs : call.dst_rs;
  a.dst_n_stride = swapped ? call.dst_rs : call.dst_cs;

  // (Sizes and depths are rounded up to tiles, and gone past by some steps, in 32 bits.)
  if (max(call.m, max(call.n, call.k)) > 0x7fffffff - 2048) return false;
  // Offsets inside a tile are 31 bits where it goes to LDS directly (fits, below, for each tile), and 32 otherwise:
  // what this leaves fits 32 in any of them, and 31 in those of 128 rows and fewer.
  const int64_t longest = (int64_t(1) << 31) / (bytes * 128) - 128;
  if (a.m.pitch > longest || a.n.pitch > longest) return false;
  const auto aligned = [&](const Side& s, Runs runs, bool dealt_rows) {
    if (reinterpret_cast<uintptr_t>(s.data) % 16 || s.pitch % granule || s.group_stride % granule) return false;
    // Runs along the depth end and, where it is dealt, begin anywhere.
    if (runs == Runs::kPlain) return columns && call.k % granule == 0;
    return !(columns && dealt_rows) && s.count % granule == 0;
  };
  const bool direct = aligned(a.m, runs_m, false) && aligned(a.n, runs_n, true);
  // Runs that the registers' way reads have 16 bytes at least.
  const auto long_enough = [&](const Side& s, Runs runs) { return (runs == Runs::kPlain ? call.k : s.count) >= granule; };
  if (!direct && !(long_enough(a.m, runs_m) && long_enough(a.n, runs_n))) return false;
  // Byte positions in a run along the depth that 32 bits do not hold, on 64x64 tiles. (Such a run is its side's only one:
  // another's pitch would be too long.)
  const bool far = !direct && (runs_m == Runs::kPlain || runs_n == Runs::kPlain) && int64_t(call.k) * bytes > 0x7fffffff - 512;
  // The tile that the CUs would be done with first. (How many tiles the groups' columns
  // make is known on the device only: here every group that can have a column ends with half a tile.)
  const int64_t busy = columns ? min(call.groups, a.n.count) : call.groups;
  const float group_depth = columns ? call.k : float(call.k) / call.groups;
  const float steps = group_depth * bytes / 128 + 0.5f + kFixedSteps;
  Grid grid;
  grid.far = far;
  int64_t blocks = 0;
  float best = 0;
  const auto fits = [&](const Side& s, Runs runs, int rows) {
    return runs == Runs::kAcross || TileOffsetsFit(rows, s.pitch * bytes, 128);
  };
  const auto step_of = [&](const TileCost& t) {
    const bool f32 = call.type == RUYAMD_DTYPE_F32;
    if (direct && !(fits(a.m, runs_m, t.m) && fits(a.n, runs_n, t.n))) return 0.0f;
    if (direct) return f32 ? t.f32 : t.direct;
    if (t.tile == Tile::k64x64) return t.through;
    if (far) return 0.0f;
    // (Both operands across the depth: 4 x 4095 x 2047, depth 8191 352 us on 64x64, 264 on 256x128, 64 x 301 x 1501, depth
    // 4001 31 and 37.)
    return f32 ? 0.0f : t.through * (columns ? 1.0f : 1.25f);
  };
  const auto most_along_n = [&](const TileCost& t) -> int64_t {
    return columns ? a.n.count / t.n + busy : ((int64_t(a.n.count) + t.n - 1) / t.n) * busy;
  };
  const auto blocks_of = [&](const TileCost& t) {
    return ((int64_t(a.m.count) + t.m - 1) / t.m * most_along_n(t) + 7) / 8 * 8;
  };
  const auto usable = [&](const TileCost& t) { return step_of(t) != 0 && LaunchFits(blocks_of(t), t.threads); };
  const auto forced = [&](const TileCost& t) { return t.m == call.forced_tile_rows && t.n == call.forced_tile_cols; };
  const bool force = std::any_of(std::begin(kTiles), std::end(kTiles), [&](const TileCost& t) { return forced(t) && usable(t); });
  for (const TileCost& t : kTiles) {
    if (!usable(t) || (force && !forced(t))) continue;
    const int64_t tiles_m = (int64_t(a.m.count) + t.m - 1) / t.m;
    const float tiles_n = columns ? std::max(float(busy), float(a.n.count) / t.n + 0.5f * busy) : most_along_n(t);
    const float rounds = std::ceil(tiles_m * tiles_n / (t.per_cu * call.compute_units) - 0.05f);
    const float time = std::max(1.0f, rounds) * steps * step_of(t);
    if (blocks == 0 || time < best) {
      best = time;
      grid.tile = t.tile;
      blocks = blocks_of(t);
    }
  }
  if (blocks == 0) return false;
  grid.blocks = static_cast<unsigned>(blocks);
  if (direct)
    LaunchType<true>(stream, a, call.type, runs_m, runs_n, grid);
  else
    LaunchType<false>(stream, a, call.type, runs_m, runs_n, grid);
  *status = hipGetLastError();
  return true;
}

}  // namespace grouped
}  // namespace ruyamd
