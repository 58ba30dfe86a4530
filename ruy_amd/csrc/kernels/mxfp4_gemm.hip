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

// kDirect: rows of both sides begin at multiples of 16 bytes and are whole blocks, so that tiles go to LDS without passing
// through registers. Otherwise rows are read 16 bytes a lane from wherever they begin.
template <int kWavesM, int kWavesN, int kBlocksM, int kBlocksN, bool kDirect>
__global__ __launch_bounds__(64 * kWavesM * kWavesN, 2) void MxFp4GemmKernel(MulCall c) {
  constexpr int kWaves = kWavesM * kWavesN;
  constexpr int kTileM = kWavesM * kBlocksM * 16, kTileN = kWavesN * kBlocksN * 16;
  // (How rows lie in LDS, which is a matter of bytes alone.)
  using M = TileSide<RUYAMD_DTYPE_BF16, Runs::kPlain, kTileM, kBlocksM, true, kWaves>;
  using N = TileSide<RUYAMD_DTYPE_BF16, Runs::kPlain, kTileN, kBlocksN, false, kWaves>;
  constexpr int kStage = M::kBytes + N::kBytes, kStages = 2;
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

  // A thread's row, whose scales it brings. (Those of rows past the tile's sides are the last row's.)
  const int row = threadIdx.x;
  const uint8_t* scale_row = c.lhs.scales;
  if (row < kTileM)
    scale_row += tile.group * c.lhs.scales_matrix_stride + int64_t(m0 + min(row, here_m - 1)) * c.lhs.scale_stride;
  else
    scale_row = c.rhs.scales + (int64_t(range.begin) + n0 + min(row - kTileM, here_n - 1)) * c.rhs.scale_stride;
  const auto fetch_scales = [&](int pair) __attribute__((always_inline)) { return LoadScales(scale_row, pair * 16, row_scales); };
  const auto put_scales = [&](const v4i& x, int pair, int buffer) __attribute__((always_inline)) {
    if (row < kRows)
      *reinterpret_cast<v4i*>(lds + kScalesAt + buffer * (kRows * 16) + row * 16) = Transposed(PlaceScales(x, pair * 16, row_scales));
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
    // As in grouped_gemm.h: steps are on their way to LDS two ahead, and the two halves of a step's depth take turns: while the
    // matrix cores have one, the fragments of the other come out of LDS. In the middle of a step all waves wait for the loads
    // of the next one and for each other; in every other step the scales of the next pair, which have come with these
    // loads, go into LDS before that, and out of it after.
    v4i next_scales = fetch_scales(0);
    issue(0, 0);
    issue(1, 1);
    put_scales(next_scales, 0, 0);
    WaitVmcnt<0>();
    Barrier();
    Fragments first, second;
    Scales scales, later;
    read(0, 0, first);
    read_scales(0, scales);
    const auto step = [&](int s, auto odd) __attribute__((always_inline)) {
      constexpr int kOdd = decltype(odd)::value;
      read(kOdd, 1, second);
      multiply(first, scales, std::integral_constant<int, 2 * kOdd>());
      interleave();
      WaitVmcnt<0>();
      if constexpr (kOdd) put_scales(next_scales, (s + 1) / 2, 0);
      Barrier();
      if constexpr (!kOdd) next_scales = fetch_scales(s / 2 + 1);
      issue(s + 2, kOdd);
      read(1 - kOdd, 0, first);
      if constexpr (kOdd) read_scales(0, later);
      multiply(second, scales, std::integral_constant<int, 2 * kOdd + 1>());
      interleave();
      if constexpr (kOdd) scales = later;
    };
    for (int s = 0;;) {
      step(s, std::integral_constant<int, 0>());
      if (++s == steps) break;
      step(s, std::integral_constant<int, 1>());
      if (++s == steps) break;
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

enum class Tile { k64x64, k128x128, k256x256 };

// A tile's sizes, the threads of its workgroup, the workgroups that a CU runs side by side, and how long one step of all of them
// takes, us, with operands straight to LDS and through registers (0: there is no such kernel).
struct TileCost {
  Tile tile;
  int m, n, threads, per_cu;
  float direct, through;
};
constexpr TileCost kTiles[] = {{Tile::k64x64, 64, 64, 256, 2, 0.48f, 0.58f},
                               {Tile::k128x128, 128, 128, 256, 2, 1.08f, 1.5f},
                               {Tile::k256x256, 256, 256, 256, 1, 1.2f, 0}};
// What a workgroup does before its first step and after its last, in steps.
constexpr float kFixedSteps = 6;

template <int kWavesM, int kWavesN, int kBlocksM, int kBlocksN, bool kDirect>
hipError_t LaunchKernel(hipStream_t stream, const MulCall& call, unsigned blocks) {
  constexpr int kRows = (kWavesM * kBlocksM + kWavesN * kBlocksN) * 16;
  constexpr int kLds = 2 * kRows * 128 + (kDirect ? 1 : 2) * kRows * 16;
  auto* const kernel = &MxFp4GemmKernel<kWavesM, kWavesN, kBlocksM, kBlocksN, kDirect>;
  static const hipError_t attribute =
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (attribute != hipSuccess) return attribute;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWavesM * kWavesN), kLds, stream, call);
  return hipGetLastError();
}

template <bool kDirect>
hipError_t LaunchTile(hipStream_t stream, const MulCall& call, Tile tile, unsigned blocks) {
  if (tile == Tile::k256x256) return LaunchLarge(stream, call, blocks);
  if (tile == Tile::k128x128) return LaunchKernel<2, 2, 4, 4, kDirect>(stream, call, blocks);
  return LaunchKernel<2, 2, 2, 2, kDirect>(stream, call, blocks);
}

}  // namespace

bool LaunchTiles(hipStream_t stream, const MulCall& call, hipError_t* status) {
  if (call.k < kBlock) return false;  // (a row has 16 bytes at least)
  // (Sizes and depths are rounded up to tiles, and gone past by some steps, in 32 bits.)
  if (std::max(call.m, std::max(call.n, call.k)) > 0x7fffffff - 2048) return false;
  const auto aligned = [&](const Matrix& m) {
    return reinterpret_cast<uintptr_t>(m.data) % 16 == 0 && m.row_bytes % 16 == 0;
  };
  const bool direct = call.k % kBlock == 0 && aligned(call.lhs) && aligned(call.rhs) && call.lhs.matrix_bytes % 16 == 0;
  // The tile that the CUs would be done with first. (How many tiles the groups' columns
  // make is known on the device only: here every group that can have a column ends with half a tile.)
  const int64_t busy = std::min(call.groups, call.n);
  const float steps = float(call.k) / kStep + 0.5f + kFixedSteps;
  const auto scales_aligned = [&](const Matrix& m) {
    return reinterpret_cast<uintptr_t>(m.scales) % 4 == 0 && m.scale_stride % 4 == 0;
  };
  const bool large = direct && call.k % 128 == 0 && call.k >= 512 && scales_aligned(call.lhs) && scales_aligned(call.rhs) &&
                     call.lhs.scales_matrix_stride % 4 == 0 && TileOffsetsFit(256, call.lhs.row_bytes, call.lhs.row_bytes) &&
                     TileOffsetsFit(256, call.rhs.row_bytes, call.rhs.row_bytes) &&
                     TileOffsetsFit(256, call.lhs.scale_stride, call.lhs.scale_stride) &&
                     TileOffsetsFit(256, call.rhs.scale_stride, call.rhs.scale_stride);
  const auto step_of = [&](const TileCost& t) {
    if (t.tile == Tile::k256x256) return large ? t.direct : 0.0f;
    if (direct && TileOffsetsFit(t.m, call.lhs.row_bytes, 128) && TileOffsetsFit(t.n, call.rhs.row_bytes, 128)) return t.direct;
    return direct ? 0.0f : t.through;
  };
  const auto blocks_of = [&](const TileCost& t) {
    return ((int64_t(call.m) + t.m - 1) / t.m * (call.n / t.n + busy) + 7) / 8 * 8;
  };
  const auto usable = [&](const TileCost& t) { return step_of(t) != 0 && LaunchFits(blocks_of(t), t.threads); };
  const auto forced = [&](const TileCost& t) { return t.m == call.forced_tile_rows && t.n == call.forced_tile_cols; };
  const bool force = std::any_of(std::begin(kTiles), std::end(kTiles), [&](const TileCost& t) { return forced(t) && usable(t); });
  Tile tile = Tile::k64x64;
  int64_t blocks = 0;
  float best = 0;
  for (const TileCost& t : kTiles) {
    if (!usable(t) || (force && !forced(t))) continue;
    const int64_t tiles_m = (int64_t(call.m) + t.m - 1) / t.m;
    const float tiles_n = std::max(float(busy), float(call.n) / t.n + 0.5f * busy);
    const float rounds = std::ceil(tiles_m * tiles_n / (t.per_cu * call.compute_units) - 0.05f);
    const float time = std::max(1.0f, rounds) * steps * step_of(t);
    if (blocks == 0 || time < best) {
      best = time;
      tile = t.tile;
      blocks = blocks_of(t);
    }
  }
  if (blocks == 0) return false;
  *status = direct ? LaunchTile<true>(stream, call, tile, static_cast<unsigned>(blocks))
                   : LaunchTile<false>(stream, call, tile, static_cast<unsigned>(blocks));
  return true;
}

}  // namespace mxfp4
}  // namespace ruyamd
