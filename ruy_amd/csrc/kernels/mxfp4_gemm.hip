// Products of 4-bit values on tiles of the destination, on the matrix cores.
//
// A workgroup makes one tile of one group's product. Both operands run along the depth and come in steps of
// 128 bytes of a row (256 values) through LDS, as those of grouped_gemm.h do; a fragment of 16
// bytes to a lane is 128 values of depth here. Scales go with them in pairs of steps, 16 bytes of a row at a time,
// transposed on their way into LDS (mxfp4_device.h), so that a fragment's scales of two steps are one word.
#include "grouped_gemm.h"
#include "launch_geometry.h"
#include "mxfp4_device.h"
#include "mxfp4_large.h"
#include "mxfp4_write_back.h"

#include <algorithm>
#include <cmath>
#include <iterator>

namespace ruyamd {
namespace mxfp4 {
namespace {

using grouped::Barrier;
using grouped::FindTile;
using grouped::kNothing;
using grouped::LoadToLds;
using grouped::Range;
using grouped::Resource;
using grouped::Runs;
using grouped::StaticFor;
using grouped::TileOf;
using grouped::TileSide;
using grouped::WaitVmcnt;

constexpr int kStep = 8 * kBlock;  // depth positions to a step: 128 bytes

// kDirect: rows of both sides begin at multiples of 4 bytes, which is what a load to LDS asks of an address, and are whole blocks, so
// that tiles go to LDS without passing through registers. (8192 x 8192 x 8192, rows 4100 bytes apart: 263 us, through registers
// 406; 4096 and 4112 apart 245 and 260.) Otherwise rows are read 16 bytes a lane from wherever they begin: 8192 x 8192 x
// 8192, rows 4097 bytes apart 496 us. (Reading the five words that hold 16 bytes and shifting them takes 503, and 8 % longer at
// 4096 x 4096 x 4096.)
// kStages: steps on their way to LDS (kDirect). More than two: the scales of the whole depth are put into LDS first, for whose
// loads the waves would otherwise wait, and for those of all steps with them, in every other step.
template <int kWavesM, int kWavesN, int kBlocksM, int kBlocksN, bool kDirect, int kStages>
__global__ __launch_bounds__(64 * kWavesM * kWavesN, 2) void MxFp4GemmKernel(MulCall c) {
  constexpr int kWaves = kWavesM * kWavesN;
  constexpr int kTileM = kWavesM * kBlocksM * 16, kTileN = kWavesN * kBlocksN * 16;
  // (How rows lie in LDS, which is a matter of bytes alone.)
  using M = TileSide<RUYAMD_DTYPE_BF16, Runs::kPlain, kTileM, kBlocksM, true, kWaves>;
  using N = TileSide<RUYAMD_DTYPE_BF16, Runs::kPlain, kTileN, kBlocksN, false, kWaves>;
  constexpr int kStage = M::kBytes + N::kBytes;
  constexpr bool kAllScales = kStages > 2;
  static_assert(kDirect || kStages == 2, "");
  constexpr int kRows = kTileM + kTileN, kScalesAt = kStages * kStage;
  static_assert(kRows <= 64 * kWaves, "a row's scales to a thread");
  using Out = WriteBack<kBlocksM, kBlocksN>;
  static_assert(kWaves * Out::kLds <= kScalesAt, "");
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave % kWavesM, wave_n = wave / kWavesM;
  const int tiles_m = (c.m + kTileM - 1) / kTileM;
  TileOf tile;
  Range range;
  if (!FindTile(c.offsets, c.groups, c.n, kTileN, tiles_m, &tile, &range)) return;
  const int m0 = tile.m * kTileM, n0 = tile.n * kTileN;
  const int here_m = min(kTileM, c.m - m0), here_n = min(kTileN, range.count - n0);
  const int steps = (c.k + kStep - 1) / kStep;
  const int row_bytes = (c.k + 1) / 2, row_scales = (c.k + kBlock - 1) / kBlock;
  const uint8_t* const base_m = c.lhs.data + tile.group * c.lhs.matrix_bytes + m0 * c.lhs.row_bytes;
  const uint8_t* const base_n = c.rhs.data + (int64_t(range.begin) + n0) * c.rhs.row_bytes;

  v4f acc[kBlocksM][kBlocksN] = {};
  struct Fragments {
    v4i m[kBlocksM], n[kBlocksN];
  };
  struct Scales {
    int m[kBlocksM], n[kBlocksN];
  };
  const auto read = [&](int stage, int kk, Fragments& f) __attribute__((always_inline)) {
    const char* const side_m = lds + stage * kStage;
#pragma unroll
    for (int j = 0; j < kBlocksN; ++j) f.n[j] = N::Fragment(side_m + M::kBytes, wave_n, j, kk, lane);
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i) f.m[i] = M::Fragment(side_m, wave_m, i, kk, lane);
  };
  // The bytes of a pair of steps: one to each half of either step.
  const auto read_scales = [&](int buffer, Scales& s) __attribute__((always_inline)) {
    const char* const at = lds + kScalesAt + buffer * (kRows * 16) + q * 4;
#pragma unroll
    for (int j = 0; j < kBlocksN; ++j)
      s.n[j] = *reinterpret_cast<const int*>(at + (kTileM + wave_n * N::kWaveRows + N::RowOf(j, l)) * 16);
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i)
      s.m[i] = *reinterpret_cast<const int*>(at + (wave_m * M::kWaveRows + M::RowOf(i, l)) * 16);
  };
  const auto multiply = [&](const Fragments& f, const Scales& s, auto byte) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) Mma<byte>(f.m[i], f.n[j], s.m[i], s.n[j], acc[i][j]);
  };

  // The scales of a row of either side. (Those of rows past the tile's sides are the last row's.)
  const auto scales_of_row = [&](int row) __attribute__((always_inline)) {
    return row < kTileM ? c.lhs.scales + tile.group * c.lhs.scales_matrix_stride + int64_t(m0 + min(row, here_m - 1)) * c.lhs.scale_stride
                        : c.rhs.scales + (int64_t(range.begin) + n0 + min(row - kTileM, here_n - 1)) * c.rhs.scale_stride;
  };
  const auto put_scales_of_row = [&](const v4i& x, int row, int pair, int buffer) __attribute__((always_inline)) {
    *reinterpret_cast<v4i*>(lds + kScalesAt + buffer * (kRows * 16) + row * 16) = Transposed(PlaceScales(x, pair * 16, row_scales));
  };
  // A thread brings those of one row, pair by pair.
  const uint8_t* const scale_row = scales_of_row(threadIdx.x);
  const auto fetch_scales = [&](int pair) __attribute__((always_inline)) { return LoadScales(scale_row, pair * 16, row_scales); };
  const auto put_scales = [&](const v4i& x, int pair, int buffer) __attribute__((always_inline)) {
    if (int(threadIdx.x) < kRows) put_scales_of_row(x, threadIdx.x, pair, buffer);
  };

  if constexpr (kDirect) {
    const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    uint32_t off_m[M::kLoads], off_n[N::kLoads];
    // (What lies beyond the tile's side is read from its last row: it ends up in rows of the tile that are not stored.)
#pragma unroll
    for (int n = 0; n < M::kLoads; ++n)
      off_m[n] = static_cast<uint32_t>(min(M::RunOf(n, wave, lane), here_m - 1) * c.lhs.row_bytes) + M::GranuleOf(n, wave, lane) * 16;
#pragma unroll
    for (int n = 0; n < N::kLoads; ++n)
      off_n[n] = static_cast<uint32_t>(min(N::RunOf(n, wave, lane), here_n - 1) * c.rhs.row_bytes) + N::GranuleOf(n, wave, lane) * 16;
    const auto issue = [&](int s, int stage) __attribute__((always_inline)) {
      const v4i rsrc_m = Resource(reinterpret_cast<const char*>(base_m) + int64_t(s) * 128);
      const v4i rsrc_n = Resource(reinterpret_cast<const char*>(base_n) + int64_t(s) * 128);
      const uint32_t to = __builtin_amdgcn_readfirstlane(lds_base + stage * kStage + wave * 1024);
      const int left = (c.k - s * kStep) / kBlock;  // granules
      if (left >= 8) {
#pragma unroll
        for (int n = 0; n < M::kLoads; ++n) LoadToLds(to + n * kWaves * 1024, off_m[n], rsrc_m);
#pragma unroll
        for (int n = 0; n < N::kLoads; ++n) LoadToLds(to + M::kBytes + n * kWaves * 1024, off_n[n], rsrc_n);
      } else {  // the last, partial step, and those behind it: zeros past the depth
#pragma unroll
        for (int n = 0; n < M::kLoads; ++n)
          LoadToLds(to + n * kWaves * 1024, M::GranuleOf(n, wave, lane) < left ? off_m[n] : kNothing, rsrc_m);
#pragma unroll
        for (int n = 0; n < N::kLoads; ++n)
          LoadToLds(to + M::kBytes + n * kWaves * 1024, N::GranuleOf(n, wave, lane) < left ? off_n[n] : kNothing, rsrc_n);
      }
    };
    // The reads of one half of a step between the products of the other.
    const auto interleave = [&]() __attribute__((always_inline)) {
      constexpr int kReads = kBlocksM + kBlocksN, kProducts = kBlocksM * kBlocksN;
      StaticFor<kReads>([](auto) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, kProducts / kReads > 0 ? kProducts / kReads : 1, 0);
      });
    };
    // As in grouped_gemm.h: steps are on their way to LDS kStages ahead, and the two halves of a step's depth take turns: while the
    // matrix cores have one, the fragments of the other come out of LDS. In the middle of a step all waves wait for the loads
    // of the next one and for each other. With two stages, in every other step the scales of the next pair, which have come with
    // these loads, go into LDS before that, and out of it after.
    constexpr int kLoads = M::kLoads + N::kLoads;
    v4i next_scales = {};
    if constexpr (!kAllScales) next_scales = fetch_scales(0);
    StaticFor<kStages>([&](auto d) __attribute__((always_inline)) { issue(d, d); });
    if constexpr (kAllScales) {
      constexpr int kAtOnce = 4, kThreads = 64 * kWaves;
      const int all = (steps + 1) / 2 * kRows;
      for (int i0 = threadIdx.x; i0 < all; i0 += kAtOnce * kThreads) {
        v4i x[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const int i = min(i0 + u * kThreads, all - 1);
          x[u] = LoadScales(scales_of_row(i % kRows), i / kRows * 16, row_scales);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const int i = i0 + u * kThreads;
          if (i < all) put_scales_of_row(x[u], i % kRows, i / kRows, i / kRows);
        }
      }
    } else {
      put_scales(next_scales, 0, 0);
    }
    WaitVmcnt<(kStages - 1) * kLoads>();
    Barrier();
    Fragments first, second;
    Scales scales, later;
    read(0, 0, first);
    read_scales(0, scales);
    const auto step = [&](int s, auto stage) __attribute__((always_inline)) {
      constexpr int kAt = decltype(stage)::value, kOdd = kAt % 2;
      read(kAt, 1, second);
      multiply(first, scales, std::integral_constant<int, 2 * kOdd>());
      interleave();
      WaitVmcnt<(kStages - 2) * kLoads>();
      if constexpr (kOdd && !kAllScales) put_scales(next_scales, (s + 1) / 2, 0);
      Barrier();
      if constexpr (!kOdd && !kAllScales) next_scales = fetch_scales(s / 2 + 1);
      issue(s + kStages, kAt);
      read((kAt + 1) % kStages, 0, first);
      // (Past the last pair: the last one again, of which nothing is used.)
      if constexpr (kOdd) read_scales(kAllScales ? min((s + 1) / 2, (steps - 1) / 2) : 0, later);
      multiply(second, scales, std::integral_constant<int, 2 * kOdd + 1>());
      interleave();
      if constexpr (kOdd) scales = later;
    };
    for (int s = 0;;) {
      step(s, std::integral_constant<int, 0>());
      if (++s == steps) break;
      step(s, std::integral_constant<int, 1>());
      if (++s == steps) break;
      if constexpr (kStages > 2) {
        step(s, std::integral_constant<int, 2>());
        if (++s == steps) break;
        step(s, std::integral_constant<int, 3>());
        if (++s == steps) break;
      }
    }
    WaitVmcnt<0>();
  } else {
    // A granule is read where it lies, or, where it would reach past the end of its row, from the row's last 16 bytes, and
    // put in its place then.
    struct Set {
      v4i m[M::kLoads], n[N::kLoads], scales;
    };
    Set held;
    const auto fetch = [&](int s) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < M::kLoads; ++n)
        held.m[n] = granule::LoadGranule<false>(base_m + min(M::RunOf(n, wave, lane), here_m - 1) * c.lhs.row_bytes,
                                                s * 128 + M::GranuleOf(n, wave, lane) * 16, row_bytes);
#pragma unroll
      for (int n = 0; n < N::kLoads; ++n)
        held.n[n] = granule::LoadGranule<false>(base_n + min(N::RunOf(n, wave, lane), here_n - 1) * c.rhs.row_bytes,
                                                s * 128 + N::GranuleOf(n, wave, lane) * 16, row_bytes);
      if (s % 2 == 0) held.scales = fetch_scales(s / 2);
    };
    const auto put = [&](int s, int stage) __attribute__((always_inline)) {
      if ((s + 1) * 128 >= row_bytes) {
#pragma unroll
        for (int n = 0; n < M::kLoads; ++n) {
          const int at = s * 128 + M::GranuleOf(n, wave, lane) * 16;
          held.m[n] = WithoutOddHalf(granule::PlaceGranule(held.m[n], at, row_bytes), int64_t(at) * 2, c.k);
        }
#pragma unroll
        for (int n = 0; n < N::kLoads; ++n)
          held.n[n] = granule::PlaceGranule(held.n[n], s * 128 + N::GranuleOf(n, wave, lane) * 16, row_bytes);
      }
      char* const to = lds + stage * kStage + (wave * 64 + lane) * 16;
#pragma unroll
      for (int n = 0; n < M::kLoads; ++n) *reinterpret_cast<v4i*>(to + n * kWaves * 1024) = held.m[n];
#pragma unroll
      for (int n = 0; n < N::kLoads; ++n) *reinterpret_cast<v4i*>(to + M::kBytes + n * kWaves * 1024) = held.n[n];
      if (s % 2 == 0) put_scales(held.scales, s / 2, s / 2 % 2);
    };
    fetch(0);
    Scales scales;
    const auto step = [&](int s, auto odd) __attribute__((always_inline)) {
      constexpr int kOdd = decltype(odd)::value;
      put(s, kOdd);
      __syncthreads();
      if (s + 1 < steps) fetch(s + 1);
      Fragments first, second;
      if constexpr (!kOdd) read_scales(s / 2 % 2, scales);
      read(kOdd, 0, first);
      read(kOdd, 1, second);
      multiply(first, scales, std::integral_constant<int, 2 * kOdd>());
      multiply(second, scales, std::integral_constant<int, 2 * kOdd + 1>());
    };
    for (int s = 0;;) {
      step(s, std::integral_constant<int, 0>());
      if (++s == steps) break;
      step(s, std::integral_constant<int, 1>());
      if (++s == steps) break;
    }
  }

  // (LDS is the write-back's now.)
  __syncthreads();
  const int row0 = wave_m * M::kWaveRows, column0 = wave_n * N::kWaveRows;
  Out{c, acc, lds + wave * Out::kLds, c.bias ? c.bias + tile.group * c.bias_stride + m0 + row0 : nullptr, m0 + row0,
      int64_t(range.begin) + n0 + column0, here_m - row0, here_n - column0}();
}

// The kernels: 64x64 with two and with four stages and 128x128 (above), and 256x256 (mxfp4_large.h).
enum class Tile { k64x64, k64x64Deep, k128x128, k256x256 };

// How long a kernel takes, us: with its tiles dealt to `per_cu` workgroups of every CU in rounds, the last of which costs at least
// `last` of a full one, fixed + rounds * (steps + more) * step, a step being 256 positions of depth. Fitted to 290 shapes of 256 to
// 16384 rows, 48 to 8192 columns and depths of 512 to 16384, bfloat16 destinations, to 5 to 11 % root mean square. Choosing by it
// costs 1.3 % over the fastest kernel at each of these shapes (20 % at the worst, 256 x 48, depth 512: 5.6 us for 4.6).
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
constexpr TileCost kTiles[] = {{Tile::k64x64, 64, 64, {4, 2.8f, 0.96f, 2.7f, 0.33f}, {2, 2.5f, 0.715f, 1.2f, 0.71f}},
                               {Tile::k64x64Deep, 64, 64, {1, 3.2f, 0.315f, 3.6f, 0.88f}, {1, 0, 0, 0, 0}},
                               {Tile::k128x128, 128, 128, {2, 2.3f, 1.34f, 3.1f, 0.51f}, {1, 3.8f, 1.24f, 0.5f, 0.90f}},
                               {Tile::k256x256, 256, 256, {1, 2.75f, 1.64f, 5.6f, 0.63f}, {1, 0, 0, 0, 0}}};

// LDS that a workgroup may take, and what 64x64 tiles of four stages do.
constexpr int kMostLds = 156 << 10;
int64_t DeepLds(int64_t k) { return 4 * 128 * 128 + (k + kChunk - 1) / kChunk * (128 * 16); }

template <int kWavesM, int kWavesN, int kBlocksM, int kBlocksN, bool kDirect, int kStages = 2>
hipError_t LaunchKernel(hipStream_t stream, const MulCall& call, unsigned blocks) {
  constexpr int kRows = (kWavesM * kBlocksM + kWavesN * kBlocksN) * 16;
  const int lds = kStages > 2 ? static_cast<int>(DeepLds(call.k)) : 2 * kRows * 128 + (kDirect ? 1 : 2) * kRows * 16;
  auto* const kernel = &MxFp4GemmKernel<kWavesM, kWavesN, kBlocksM, kBlocksN, kDirect, kStages>;
  static const hipError_t attribute =
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
  if (attribute != hipSuccess) return attribute;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWavesM * kWavesN), lds, stream, call);
  return hipGetLastError();
}

template <bool kDirect>
hipError_t LaunchTile(hipStream_t stream, const MulCall& call, Tile tile, unsigned blocks) {
  if (tile == Tile::k256x256) return LaunchLarge(stream, call, blocks);
  if constexpr (kDirect)
    if (tile == Tile::k64x64Deep) return LaunchKernel<2, 2, 2, 2, true, 4>(stream, call, blocks);
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
  const auto scales_aligned = [&](const Matrix& m) {
    return reinterpret_cast<uintptr_t>(m.scales) % 4 == 0 && m.scale_stride % 4 == 0;
  };
  const bool large = direct && call.k % 128 == 0 && call.k >= 512 && scales_aligned(call.lhs) && scales_aligned(call.rhs) &&
                     call.lhs.scales_matrix_stride % 4 == 0 && TileOffsetsFit(256, call.lhs.row_bytes, call.lhs.row_bytes) &&
                     TileOffsetsFit(256, call.rhs.row_bytes, call.rhs.row_bytes) &&
                     TileOffsetsFit(256, call.lhs.scale_stride, call.lhs.scale_stride) &&
                     TileOffsetsFit(256, call.rhs.scale_stride, call.rhs.scale_stride);
  const auto fits = [&](const TileCost& t) {
    return TileOffsetsFit(t.m, call.lhs.row_bytes, 128) && TileOffsetsFit(t.n, call.rhs.row_bytes, 128);
  };
  const auto timing_of = [&](const TileCost& t) {
    const Timing none = {1, 0, 0, 0, 0};
    if (t.tile == Tile::k256x256) return large ? t.direct : none;
    if (t.tile == Tile::k64x64Deep && DeepLds(call.k) > kMostLds) return none;
    return !direct ? t.through : fits(t) ? t.direct : none;
  };
  const int64_t busy = std::min(call.groups, call.n);
  const auto blocks_of = [&](const TileCost& t) {
    return ((int64_t(call.m) + t.m - 1) / t.m * (call.n / t.n + busy) + 7) / 8 * 8;
  };
  const auto usable = [&](const TileCost& t) { return timing_of(t).step != 0 && LaunchFits(blocks_of(t), kThreads); };
  const auto forced = [&](const TileCost& t) {
    return t.m == call.forced_tile_rows && t.n == call.forced_tile_cols && (t.tile == Tile::k64x64Deep) == call.forced_deep;
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
    const float rounds = std::max(timing.last, full + (all > full ? timing.last + (1 - timing.last) * (all - full) : 0.0f));
    const float time = timing.fixed + rounds * (float(call.k) / kStep + timing.more) * timing.step;
    if (choice.blocks == 0 || time < choice.time) {
      choice.time = time;
      choice.tile = t.tile;
      choice.blocks = blocks_of(t);
    }
  }
  // Weights out of HBM, one matrix and one to each group.
  const double bytes = double(busy) * call.m * (call.lhs.row_bytes + call.lhs.scale_stride);
  choice.time = std::max(choice.time, 3.0f + static_cast<float>(bytes / (busy == 1 ? 3.9e6 : 4.5e6)));
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
