// Products of 4-bit values on tiles of the destination, on the matrix cores.
//
// A workgroup makes one tile of one group's product. Both operands run along the depth and come in steps of
// 128 bytes of a row (256 values) through LDS, as those of grouped_gemm.h do; a fragment of 16
// bytes to a lane is 128 values of depth here. Scales go with them in pairs of steps, 16 bytes of a row at a time,
// transposed on their way into LDS (mxfp4_device.h), so that a fragment's scales of two steps are one word.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 cycles with 4-bit values on both sides, so a wave's step of 64x64 is 512 cycles of products, of 16 KB
// out of LDS (a CU's four waves 512 cycles) and of 8 KB into it; a tile waits for what is not done beside its products. Few
// tiles: four stages, and one workgroup to a CU (2048 x 2048 x 8192: 128x128 26 to 28 us, 2.4 to 2.6 PFLOP/s; with two stages 30.5; the
// matrix cores are busy in a third of a deeper product's cycles, and waves wait in 29 %). Many:
// two workgroups of 128x128 to a CU, one of which multiplies while the other waits (2048 x 4096 x 4096, forced, 25.0 us, with
// four stages 29.5), of 256x128 (mxfp4_wide.hip; 16384 x 3300 x 512 35.0 us, 128x128 49.5), or 256x256, which read half as much for a
// product (4096 x 4096 x 4096 37.3 us, 128x128 46).
#include "launch_geometry.h"
#include "mxfp4_large.h"
#include "mxfp4_tile.h"

#include <algorithm>
#include <cmath>
#include <iterator>

namespace ruyamd {
namespace mxfp4 {
namespace {

template <int kWavesM, int kWavesN, int kBlocksM, int kBlocksN, bool kDirect, int kStages, ScaleLoads kScaleLoads>
__global__ __launch_bounds__(64 * kWavesM * kWavesN, 2) void MxFp4GemmKernel(MulCall c) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int kTileM = kWavesM * kBlocksM * 16, kTileN = kWavesN * kBlocksN * 16;
  TileOf tile;
  Range range;
  if (!FindTile(c.offsets, c.groups, c.n, kTileN, (c.m + kTileM - 1) / kTileM, &tile, &range)) return;
  MultiplyTile<kWavesM, kWavesN, kBlocksM, kBlocksN, kDirect, kStages, kScaleLoads>(c, tile, range, lds);
}

// The kernels: 64x64 and 128x128 with two and with four stages (mxfp4_tile.h), 256x128 and 256x256 (mxfp4_large.h).
enum class Tile { k64x64, k64x64Deep, k128x128, k128x128Deep, k256x128, k256x256 };
bool IsDeep(Tile t) { return t == Tile::k64x64Deep || t == Tile::k128x128Deep; }

// How long a kernel takes, us: with its tiles dealt to `per_cu` workgroups of every CU in rounds, the last of which costs at least
// `last` of a full one, fixed + rounds * (steps + more) * step, a step being 256 positions of depth; a quarter of a round or less
// of 256x256 tiles behind full ones, which is made in quarters, (steps + kQuarters.more) * kQuarters.step. Fitted to 551 shapes of 256 to
// 16384 rows, 48 to 8192 columns and depths of 512 to 8192, bfloat16 destinations, to 5 to 10 % root mean square. Choosing by it
// costs 0.9 % over the fastest kernel at each of these shapes (16 % at the worst, 256 x 6000, depth 4096: 12.0 us for 10.4). Of sizes
// that are not among them, 2048 x 4096 x 4096 goes to 256x128 and takes 29.5 us for the 25.0 of 128x128.
struct Timing {
  int per_cu;
  float fixed, step, more, last;
};
struct TileCost {
  Tile tile;
  int m, n;
  Timing direct, through;  // operands straight to LDS, and through registers (step 0: there is no such kernel)
};
constexpr int kThreads = 256;
constexpr TileCost kTiles[] = {{Tile::k64x64, 64, 64, {4, 3.0f, 0.943f, 2.6f, 0.31f}, {2, 2.7f, 0.702f, 1.2f, 0.67f}},
                               {Tile::k64x64Deep, 64, 64, {1, 3.2f, 0.236f, 5.8f, 0.87f}, {1, 0, 0, 0, 0}},
                               {Tile::k128x128, 128, 128, {2, 3.2f, 1.21f, 3.35f, 0.39f}, {1, 4.1f, 1.22f, 0.38f, 0.90f}},
                               {Tile::k128x128Deep, 128, 128, {1, 2.45f, 0.628f, 6.4f, 0.72f}, {1, 0, 0, 0, 0}},
                               {Tile::k256x128, 256, 128, {1, 4.0f, 1.26f, 1.5f, 0.72f}, {1, 0, 0, 0, 0}},
                               {Tile::k256x256, 256, 256, {1, 3.6f, 1.66f, 5.15f, 0.63f}, {1, 0, 0, 0, 0}}};
constexpr struct {
  float step, more;
} kQuarters = {0.58f, 6.4f};

// LDS that a workgroup may take, and what 64x64 tiles of four stages do.
constexpr int kMostLds = 156 << 10;
int64_t DeepLds(int64_t k) { return 4 * 128 * 128 + (k + kChunk - 1) / kChunk * (128 * 16); }

template <int kWavesM, int kWavesN, int kBlocksM, int kBlocksN, bool kDirect, int kStages = 2,
          ScaleLoads kScaleLoads = ScaleLoads::kThroughRegisters>
hipError_t LaunchKernel(hipStream_t stream, const MulCall& call, unsigned blocks) {
  constexpr int kRows = (kWavesM * kBlocksM + kWavesN * kBlocksN) * 16;
  const int lds = kScaleLoads == ScaleLoads::kAllFirst     ? static_cast<int>(DeepLds(call.k))
                  : kScaleLoads == ScaleLoads::kAhead      ? kStages * kRows * 128 + 3 * kRows * 16
                  : kScaleLoads == ScaleLoads::kAheadWords ? kStages * kRows * 128 + kRows * 16 + 2 * kRows * 20
                                                           : kStages * kRows * 128 + (kDirect ? 1 : 2) * kRows * 16;
  auto* const kernel = &MxFp4GemmKernel<kWavesM, kWavesN, kBlocksM, kBlocksN, kDirect, kStages, kScaleLoads>;
  static const hipError_t attribute =
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
  if (attribute != hipSuccess) return attribute;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWavesM * kWavesN), lds, stream, call);
  return hipGetLastError();
}

template <bool kDirect>
hipError_t LaunchTile(hipStream_t stream, const MulCall& call, Tile tile, unsigned blocks) {
  if (tile == Tile::k256x256) return LaunchLarge(stream, call, blocks);
  if (tile == Tile::k256x128) return LaunchWide(stream, call, blocks);
  if constexpr (kDirect)
    if (tile == Tile::k64x64Deep) return LaunchKernel<2, 2, 2, 2, true, 4, ScaleLoads::kAllFirst>(stream, call, blocks);
  if constexpr (kDirect)
    if (tile == Tile::k128x128Deep)
      return ScalesNeedWords(call) ? LaunchKernel<2, 2, 4, 4, true, 4, ScaleLoads::kAheadWords>(stream, call, blocks)
                                   : LaunchKernel<2, 2, 4, 4, true, 4, ScaleLoads::kAhead>(stream, call, blocks);
  if (tile == Tile::k128x128) return LaunchKernel<2, 2, 4, 4, kDirect>(stream, call, blocks);
  return LaunchKernel<2, 2, 2, 2, kDirect>(stream, call, blocks);
}

// The tiles of a call, how many at most, and how long they take (blocks 0: none are its).
struct Choice {
  Tile tile = Tile::k64x64;
  bool direct = false;
  int64_t blocks = 0;
  float time = 0;
};

Choice Choose(const MulCall& call) {
  Choice choice;
  if (call.k < kBlock) return choice;  // (a row has 16 bytes at least)
  // (Sizes and depths are rounded up to tiles, and gone past by some steps, in 32 bits.)
  if (std::max(call.m, std::max(call.n, call.k)) > 0x7fffffff - 2048) return choice;
  const auto aligned = [&](const Matrix& m) {
    return reinterpret_cast<uintptr_t>(m.data) % 4 == 0 && m.row_bytes % 4 == 0;
  };
  const bool direct = call.k % kBlock == 0 && aligned(call.lhs) && aligned(call.rhs) && call.lhs.matrix_bytes % 4 == 0;
  const bool large = direct && call.k >= 512 && TileOffsetsFit(256, call.lhs.row_bytes, call.lhs.row_bytes) &&
                     TileOffsetsFit(256, call.rhs.row_bytes, call.rhs.row_bytes) &&
                     TileOffsetsFit(256, call.lhs.scale_stride, call.lhs.scale_stride + 4) &&
                     TileOffsetsFit(256, call.rhs.scale_stride, call.rhs.scale_stride + 4);
  const auto fits = [&](const TileCost& t) {
    return TileOffsetsFit(t.m, call.lhs.row_bytes, call.lhs.row_bytes) && TileOffsetsFit(t.n, call.rhs.row_bytes, call.rhs.row_bytes);
  };
  const auto timing_of = [&](const TileCost& t) {
    const Timing none = {1, 0, 0, 0, 0};
    if (t.tile == Tile::k256x256 || t.tile == Tile::k256x128 || t.tile == Tile::k128x128Deep) return large ? t.direct : none;
    if (t.tile == Tile::k64x64Deep && DeepLds(call.k) > kMostLds) return none;
    return !direct ? t.through : fits(t) ? t.direct : none;
  };
  const int64_t busy = std::min(call.groups, call.n);
  const auto blocks_of = [&](const TileCost& t) {
    const int64_t tiles_m = (int64_t(call.m) + t.m - 1) / t.m;
    const int64_t tiles = call.offsets ? tiles_m * (call.n / t.n + busy) : tiles_m * ((int64_t(call.n) + t.n - 1) / t.n);
    // (Of the largest tiles three more workgroups for each that may go to quarters.)
    const int64_t each_xcd = (tiles + 7) / 8;
    if (t.tile != Tile::k256x256) return each_xcd * 8;
    return XcdWorkgroups(each_xcd, TilesAtOnce(call.compute_units), call.offsets != nullptr) * 8;
  };
  const auto usable = [&](const TileCost& t) { return timing_of(t).step != 0 && LaunchFits(blocks_of(t), kThreads); };
  const auto forced = [&](const TileCost& t) {
    return t.m == call.forced_tile_rows && t.n == call.forced_tile_cols && IsDeep(t.tile) == call.forced_deep;
  };
  const bool force = std::any_of(std::begin(kTiles), std::end(kTiles), [&](const TileCost& t) { return forced(t) && usable(t); });
  // The kernel that would be done first. (How many tiles the groups' columns make is known on the device only: here every group that can
  // have a column ends with half a tile.)
  choice.direct = direct;
  for (const TileCost& t : kTiles) {
    if (!usable(t) || (force && !forced(t))) continue;
    const Timing timing = timing_of(t);
    const int64_t tiles_m = (int64_t(call.m) + t.m - 1) / t.m;
    const float tiles_n = busy == 1 ? std::ceil(float(call.n) / t.n) : std::max(float(busy), float(call.n) / t.n + 0.5f * busy);
    const float all = tiles_m * tiles_n / (timing.per_cu * call.compute_units), full = std::floor(all);
    const float steps = float(call.k) / kStep;
    const bool quarters = t.tile == Tile::k256x256 && full >= 1 && all > full && all - full <= 0.25f;
    const float rounds =
        quarters ? full : std::max(timing.last, full + (all > full ? timing.last + (1 - timing.last) * (all - full) : 0.0f));
    const float time = timing.fixed + rounds * (steps + timing.more) * timing.step +
                       (quarters ? (steps + kQuarters.more) * kQuarters.step : 0.0f);
    if (choice.blocks == 0 || time < choice.time) {
      choice.time = time;
      choice.tile = t.tile;
      choice.blocks = blocks_of(t);
    }
  }
  // Weights out of HBM, one matrix and one to each group.
  const double bytes = double(busy) * call.m * (call.lhs.row_bytes + call.lhs.scale_stride);
  choice.time = std::max(choice.time, 2.6f + static_cast<float>(bytes / (busy == 1 ? 4.6e6 : 5.0e6)));
  return choice;
}

}  // namespace

float TilesMicroseconds(const MulCall& call) {
  const Choice choice = Choose(call);
  return choice.blocks ? choice.time : -1;
}

bool LaunchTiles(hipStream_t stream, const MulCall& call, hipError_t* status) {
  const Choice choice = Choose(call);
  if (choice.blocks == 0) return false;
  const unsigned blocks = static_cast<unsigned>(choice.blocks);
  *status = choice.direct ? LaunchTile<true>(stream, call, choice.tile, blocks) : LaunchTile<false>(stream, call, choice.tile, blocks);
  return true;
}

}  // namespace mxfp4
}  // namespace ruyamd
