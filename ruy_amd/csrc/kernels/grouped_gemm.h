// Grouped products on tiles of the destination, on the matrix cores.
//
// A workgroup makes one tile of one group's product: kTileM x kTileN elements,
// the M side the one along which the destination is contiguous. Each operand
// comes in steps of 128 bytes of depth (64 values of 16 bits, 32 of 32) through
// LDS, in the order in which it lies in memory: runs along the depth (kPlain) or
// along the tile's side (kAcross, such as the weights in a token gradient and both
// operands of a weight gradient). Fragments of the latter come out of LDS through
// the transposing reads of gfx950, so no operand is ever copied for its order.
//
// What bounds it where there are many tiles: steps reach LDS out of L2 at 10 to 12 TB/s over the
// card, of which 256x256 needs a quarter of 64x64's bytes and is the best tile wherever there are
// enough of them; and the last round of tiles, of which a part of the CUs has none. bfloat16, 8 groups of 4096x2048
// by 8192 columns: 162 us, 850 TFLOP/s (one library product of that work 115 us, a floor of 95 at the rate of a
// large one), 576 tiles on 256 CUs; with groups of one size, 512 tiles, a tenth less. Where the depth is dealt, tiles go
// to the XCDs by their number and not by their depth: 8 weight gradients of 2048x4096 over 8192 columns, fp32, 187 us with
// groups of one size, 227, 263 and 361 where group i has a share of (i + 1) ^ -0.25, -0.5 and -1. Where depths
// are short (half, 48 weight gradients of 515x771, depth 2500 in all, 40 us) it is the
// latency of a tile's few steps and its write-back. fp32 runs on the matrix cores' own fp32
// instructions: 4 groups of 1024x1024 by 1500 columns 36 us, 88 TFLOP/s of 143.
#ifndef RUY_AMD_CSRC_KERNELS_GROUPED_GEMM_H_
#define RUY_AMD_CSRC_KERNELS_GROUPED_GEMM_H_

#include <hip/hip_runtime.h>

#include <type_traits>
#include <utility>

#include "granule.h"
#include "grouped_device.h"

namespace ruyamd {
namespace grouped {

using granule::v4i;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

enum class Runs { kPlain, kAcross };

// One side of the product as a workgroup's tile sees it.
struct Side {
  const void* data = nullptr;
  int64_t pitch = 0;         // values from a run to the next
  int64_t group_stride = 0;  // values from a group's matrix to the next one's
  int count = 0;             // rows (columns) of the side, over all groups where they are dealt
};

struct GemmArgs {
  Dealt dealt;
  Side m, n;
  void* dst;
  int64_t dst_m_stride, dst_n_stride, dst_group_stride;
  const int32_t* offsets;
  int groups, depth;  // depth: over all groups where it is dealt
  const float* bias;  // one value to each place of the M side
  int64_t bias_stride;
  float clamp_min, clamp_max;
  int dst_f32;
};

// f(std::integral_constant<int, 0>()), ..., f(std::integral_constant<int, N - 1>()).
template <class F, int... Is>
__device__ __forceinline__ void StaticForEach(F&& f, std::integer_sequence<int, Is...>) {
  (f(std::integral_constant<int, Is>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void StaticFor(F&& f) {
  StaticForEach(f, std::make_integer_sequence<int, N>());
}

// 64 lanes x 16 bytes from the lanes' offsets to 1024 bytes of LDS, on their way
// until vmcnt says otherwise. Offsets at or past the end of `rsrc` bring zeros.
__device__ __forceinline__ void LoadToLds(uint32_t lds, uint32_t voffset, v4i rsrc) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(lds), "v"(voffset), "s"(rsrc)
      : "memory");
}
template <int N>
__device__ __forceinline__ void WaitVmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void Barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// What a lane's offset is set to for zeros; offsets inside a tile stay below it.
constexpr uint32_t kNothing = 0x80000000u;
__device__ __forceinline__ v4i Resource(const char* base) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  v4i r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(a & 0xffffffffu));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<int>((a >> 32) & 0xffffu));
  r[2] = static_cast<int>(kNothing);
  r[3] = 0x00020000;
  return r;
}

template <int kType>
struct Element {
  static constexpr int kBytes = kType == RUYAMD_DTYPE_F32 ? 4 : 2;
  static constexpr int kDepth = 128 / kBytes;     // depth positions to a step
  static constexpr int kGranule = 16 / kBytes;    // values to 16 bytes
};

// Two fragments of 16 bytes: 16 rows x 16 columns x 4 granules of depth.
template <int kType>
__device__ __forceinline__ void Mma(const v4i& a, const v4i& b, v4f& acc) {
  if constexpr (kType == RUYAMD_DTYPE_BF16) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), acc, 0, 0, 0);
  } else if constexpr (kType == RUYAMD_DTYPE_F16) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(a[e]), __int_as_float(b[e]), acc, 0, 0, 0);
  }
}

// One side of the tile: how it is laid out in LDS, loaded and read. `kRows` rows
// of the tile in `kWaveRows`-row pieces, one to a wave, of kBlocks blocks of 16.
template <int kType, Runs kRuns, int kTileRows, int kBlocks, bool kPermuted, int kWaves>
struct TileSide {
  using E = Element<kType>;
  static constexpr int kRows = kTileRows;
  static constexpr int kBytes = kRows * 128;                 // in LDS, per step
  static constexpr int kLoads = kBytes / 1024 / kWaves;      // per wave and step
  static constexpr int kRunGranules = kRuns == Runs::kPlain ? 8 : kRows / E::kGranule;
  static constexpr int kRunsPerLoad = 64 / kRunGranules;     // (0: a run takes several loads)
  static constexpr int kWaveRows = 16 * kBlocks;
  static constexpr int kReads = kRuns == Runs::kPlain ? 1 : E::kBytes == 2 ? 2 : 4;  // of LDS, for a fragment
  static_assert(kBytes % (1024 * kWaves) == 0, "");

  // Row of the wave's piece that lane l (mod 16) holds of block b. Where the rows
  // are permuted, a lane's accumulators of two blocks are of 8 consecutive ones.
  static __device__ __forceinline__ int RowOf(int b, int l) {
    return kPermuted ? (b >> 1) * 32 + (l >> 2) * 8 + (b & 1) * 4 + (l & 3) : b * 16 + l;
  }

  // Granule g of run r is stored in slot g ^ Key(r): lanes that read LDS together
  // then reach all banks.
  static __device__ __forceinline__ int Key(int r) {
    if constexpr (kRuns == Runs::kPlain) {
      if constexpr (kPermuted) return ((r >> 1) & 1) | ((r >> 3) & 3) << 1;
      return (r >> 1) & 7;
    } else if constexpr (E::kBytes == 2) {
      // Reads of 4 consecutive runs of each of 4 groups of 8, 32 bytes of each.
      return (((r & 3) | ((r >> 3) & 3) << 2) << 1) & (kRunGranules - 1);
    } else {
      return (r >> 2) & 3;
    }
  }

  // Where load number n of a wave puts what lane `lane` brings: run and granule.
  static __device__ __forceinline__ int RunOf(int n, int wave, int lane) {
    return ((n * kWaves + wave) * 64 + lane) / kRunGranules;
  }
  static __device__ __forceinline__ int GranuleOf(int n, int wave, int lane) {
    return (((n * kWaves + wave) * 64 + lane) % kRunGranules) ^ Key(RunOf(n, wave, lane));
  }

  // The fragment of block b and depth half kk (0, 1) from the side's LDS; `piece`: the wave's.
  static __device__ __forceinline__ v4i Fragment(const char* lds, int piece, int b, int kk, int lane) {
    const int l = lane & 15, q = lane >> 4;
    if constexpr (kRuns == Runs::kPlain) {
      const int r = piece * kWaveRows + RowOf(b, l);
      return *reinterpret_cast<const v4i*>(lds + r * 128 + (((kk * 4 + q) ^ Key(r)) << 4));
    } else if constexpr (E::kBytes == 2) {
      // (A read hands lane l of 16 the l-th column of the 4 runs x 16 values
      // that the 16 lanes point at, 4 values each.)
      v4s half[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int run = kk * 32 + q * 8 + h * 4 + (l >> 2);
        const int at = piece * kWaveRows + RowOf(b, (l & 3) * 4);
        const char* p = lds + run * (kRows * 2) + (((at >> 3) ^ Key(run)) << 4) + (at & 7) * 2;
        half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p);
      }
      return __builtin_bit_cast(v4i, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      v4i f;
      const int at = piece * kWaveRows + RowOf(b, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int run = kk * 16 + q * 4 + e;
        f[e] = *reinterpret_cast<const int*>(lds + run * (kRows * 4) + (((at >> 2) ^ Key(run)) << 4) + (at & 3) * 4);
      }
      return f;
    }
  }
};

// Two values rounded to a 16-bit type, in one register.
template <int kType>
__device__ __forceinline__ int RoundPair(float x, float y) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f both = {x, y};
  if constexpr (kType == RUYAMD_DTYPE_BF16) {
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(int, __builtin_convertvector(both, v2bf));
  } else {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(int, __builtin_convertvector(both, v2h));
  }
}

// The range of a group that is the same for the whole wave, in scalar registers.
__device__ __forceinline__ Range UniformRangeOf(const int32_t* offsets, int group, int total) {
  const Range r = RangeOf(offsets, group, total);
  return {__builtin_amdgcn_readfirstlane(r.begin), __builtin_amdgcn_readfirstlane(r.count)};
}

// The tile a workgroup makes: its group, and which along either side.
struct TileOf {
  int group, m, n;
};

// The sum of the lanes' values up to and with each lane's own.
__device__ __forceinline__ int InclusiveSum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // from 1, 2, 4, 8 lanes below in its row of 16,
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);  // the last lane of row 0 (2) to row 1 (3),
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);  // of row 1 to rows 2 and 3
  return v;
}

// Tiles of groups whose columns are dealt: how many a group has is known here only.
// Workgroups go round the eight XCDs one by one; each XCD gets a contiguous
// run of the tiles, so that what its L2 holds serves several of them. Tiles of a
// group go in bands of kBand along the N side.
// (Offsets that run backwards may have every other group take all columns. 64 groups have fewer than 2^31 tiles even so, as a
// launch has fewer than 2^26 workgroups, and the search ends; their total may wrap round, and tiles are left out then.)
constexpr int kBand = 8;
__device__ __forceinline__ bool FindTile(const int32_t* offsets, int groups, int columns, int tile_n, int tiles_m,
                                         TileOf* tile, Range* range) {
  const int lane = threadIdx.x & 63;
  struct Lane {
    int begin, count, tiles;
  };
  // What lane l knows of group g0 + l.
  const auto look = [&](int g) __attribute__((always_inline)) -> Lane {
    if (g >= groups) return {0, 0, 0};
    const Range r = RangeOf(offsets, g, columns);
    return {r.begin, r.count, (r.count + tile_n - 1) / tile_n};
  };
  Lane mine = look(lane);
  int upto = InclusiveSum(mine.tiles), total = __builtin_amdgcn_readlane(upto, 63);
  if (groups > 64) {  // (the total first: the XCDs' shares go by it)
    for (int g0 = 64; g0 < groups; g0 += 64) total += __builtin_amdgcn_readlane(InclusiveSum(look(g0 + lane).tiles), 63);
  }
  // (int64_t: tiles of many groups times those of many rows.)
  const int64_t all = int64_t(total) * tiles_m, per_xcd = (all + 7) / 8;
  const int64_t place = blockIdx.x >> 3;
  const int64_t t = int64_t(blockIdx.x & 7) * per_xcd + place;
  if (place >= per_xcd || t >= all) return false;
  int64_t before = 0;
  for (int g0 = 0;;) {
    const uint64_t past = __ballot((before + upto) * tiles_m > t);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int tiles = __builtin_amdgcn_readlane(mine.tiles, at);
      const int64_t group_first = (before + __builtin_amdgcn_readlane(upto, at) - tiles) * tiles_m;
      int in_group = static_cast<int>(t - group_first);
      const int band = in_group / (kBand * tiles_m), width = min(kBand, tiles - band * kBand);
      in_group -= band * kBand * tiles_m;
      *tile = {g0 + at, in_group / width, band * kBand + in_group % width};
      *range = {__builtin_amdgcn_readlane(mine.begin, at), __builtin_amdgcn_readlane(mine.count, at)};
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    g0 += 64;
    mine = look(g0 + lane);
    upto = InclusiveSum(mine.tiles);
  }
}

// kDirect: every run of both operands begins at a multiple of 16 bytes and is a
// whole number of granules, so that tiles go to LDS without passing through
// registers. Otherwise they are read 16 bytes a lane from wherever they begin, the
// granule in which a run ends put in its place (granule.h), and written to LDS.
// kFar (not kDirect): runs along the depth may have more than 2^31 bytes, as one row or column stored value behind value
// may, such as the ones of a bias gradient.
template <int kType, Runs kRunsM, Runs kRunsN, int kWavesM, int kWavesN, int kBlocksM, int kBlocksN, bool kDirect, int kStages,
          bool kFar>
// (At least two waves to a SIMD: with more registers than that leaves it the compiler puts the accumulators into the
// second register file and moves them there and back on every step.)
__global__ __launch_bounds__(64 * kWavesM * kWavesN, 2) void GroupedGemmKernel(GemmArgs p) {
  using E = Element<kType>;
  constexpr int kWaves = kWavesM * kWavesN;
  constexpr int kTileM = kWavesM * kBlocksM * 16, kTileN = kWavesN * kBlocksN * 16;
  using M = TileSide<kType, kRunsM, kTileM, kBlocksM, kRunsM == Runs::kPlain, kWaves>;
  using N = TileSide<kType, kRunsN, kTileN, kBlocksN, false, kWaves>;
  constexpr int kStage = M::kBytes + N::kBytes;
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave % kWavesM, wave_n = wave / kWavesM;
  const int tiles_m = (p.m.count + kTileM - 1) / kTileM;

  TileOf tile;
  Range range;
  const bool columns = p.dealt == Dealt::kColumns;
  if (columns) {
    if (!FindTile(p.offsets, p.groups, p.n.count, kTileN, tiles_m, &tile, &range)) return;
  } else {
    const int tiles_n = (p.n.count + kTileN - 1) / kTileN;
    const int64_t all = int64_t(p.groups) * tiles_m * tiles_n, per_xcd = (all + 7) / 8, place = blockIdx.x >> 3;
    const int64_t t = int64_t(blockIdx.x & 7) * per_xcd + place;
    if (place >= per_xcd || t >= all) return;
    tile.group = static_cast<int>(t / (tiles_m * tiles_n));
    int in_group = static_cast<int>(t - int64_t(tile.group) * tiles_m * tiles_n);
    const int band = in_group / (kBand * tiles_m), width = min(kBand, tiles_n - band * kBand);
    in_group -= band * kBand * tiles_m;
    tile.m = in_group / width;
    tile.n = band * kBand + in_group % width;
    range = UniformRangeOf(p.offsets, tile.group, p.depth);
  }
  const int rows_m = p.m.count, rows_n = columns ? range.count : p.n.count;
  const int depth = columns ? p.depth : range.count;
  const int m0 = tile.m * kTileM, n0 = tile.n * kTileN;
  const int here_m = min(kTileM, rows_m - m0), here_n = min(kTileN, rows_n - n0);

  // The first value of each side's part of the operand.
  const auto base_of = [&](const Side& s, Runs runs, int first, bool dealt_rows) __attribute__((always_inline)) {
    int64_t at = columns ? (dealt_rows ? 0 : tile.group * s.group_stride) : 0;
    int64_t row = first, k = 0;
    if (columns && dealt_rows) row += range.begin;
    if (!columns) k = range.begin;
    at += runs == Runs::kPlain ? row * s.pitch + k : k * s.pitch + row;
    return static_cast<const char*>(s.data) + at * E::kBytes;
  };
  const char* base_m = base_of(p.m, kRunsM, m0, false);
  const char* base_n = base_of(p.n, kRunsN, n0, true);

  const int steps = (depth + E::kDepth - 1) / E::kDepth;

  v4f acc[kBlocksM][kBlocksN] = {};
  struct Fragments {
    v4i m[kBlocksM], n[kBlocksN];
  };
  const auto read = [&](int stage, int kk, Fragments& f) __attribute__((always_inline)) {
    const char* const side_m = lds + stage * kStage;
#pragma unroll
    for (int j = 0; j < kBlocksN; ++j) f.n[j] = N::Fragment(side_m + M::kBytes, wave_n, j, kk, lane);
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i) f.m[i] = M::Fragment(side_m, wave_m, i, kk, lane);
  };
  const auto multiply = [&](const Fragments& f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i)
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) Mma<kType>(f.m[i], f.n[j], acc[i][j]);
  };
  // The reads of one half of a step between the products of the other.
  const auto interleave = [&]() __attribute__((always_inline)) {
    constexpr int kReads = M::kReads * kBlocksM + N::kReads * kBlocksN;
    constexpr int kProducts = kBlocksM * kBlocksN * (E::kBytes == 4 ? 4 : 1);
    constexpr int kEach = kProducts / kReads > 0 ? kProducts / kReads : 1;
    StaticFor<(kReads < kProducts ? kReads : kProducts)>([](auto) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_group_barrier(0x100, kReads / kProducts > 0 ? kReads / kProducts : 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
    });
  };

  if constexpr (kDirect) {
    const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    uint32_t off_m[M::kLoads], off_n[N::kLoads];
    // A lane's offset of load n, and its first depth position. What lies beyond
    // the tile's side is read from the side's last row (granule): it ends up
    // in rows of the tile that are not stored.
    const auto offset_of = [&](auto side, int n, int here, Runs runs, int64_t pitch) __attribute__((always_inline)) {
      using T = decltype(side);
      const int run = T::RunOf(n, wave, lane), granule = T::GranuleOf(n, wave, lane);
      if (runs == Runs::kPlain)
        return static_cast<uint32_t>(min(run, here - 1) * pitch * E::kBytes) + granule * 16;
      return static_cast<uint32_t>(run * pitch * E::kBytes) + min(granule, here / E::kGranule - 1) * 16;
    };
    const auto depth_of = [&](auto side, int n, Runs runs) __attribute__((always_inline)) {
      using T = decltype(side);
      return runs == Runs::kPlain ? T::GranuleOf(n, wave, lane) * E::kGranule : T::RunOf(n, wave, lane);
    };
#pragma unroll
    for (int n = 0; n < M::kLoads; ++n) off_m[n] = offset_of(M(), n, here_m, kRunsM, p.m.pitch);
#pragma unroll
    for (int n = 0; n < N::kLoads; ++n) off_n[n] = offset_of(N(), n, here_n, kRunsN, p.n.pitch);
    const int64_t step_m = (kRunsM == Runs::kPlain ? 1 : p.m.pitch) * 128;
    const int64_t step_n = (kRunsN == Runs::kPlain ? 1 : p.n.pitch) * 128;
    const auto issue = [&](int s, int stage) __attribute__((always_inline)) {
      const v4i rsrc_m = Resource(base_m + s * step_m), rsrc_n = Resource(base_n + s * step_n);
      const uint32_t to = __builtin_amdgcn_readfirstlane(lds_base + stage * kStage + wave * 1024);
      const int left = depth - s * E::kDepth;
      if (left >= E::kDepth) {
#pragma unroll
        for (int n = 0; n < M::kLoads; ++n) LoadToLds(to + n * kWaves * 1024, off_m[n], rsrc_m);
#pragma unroll
        for (int n = 0; n < N::kLoads; ++n) LoadToLds(to + M::kBytes + n * kWaves * 1024, off_n[n], rsrc_n);
      } else {  // the last, partial step, and those behind it: zeros past the depth
#pragma unroll
        for (int n = 0; n < M::kLoads; ++n)
          LoadToLds(to + n * kWaves * 1024, depth_of(M(), n, kRunsM) < left ? off_m[n] : kNothing, rsrc_m);
#pragma unroll
        for (int n = 0; n < N::kLoads; ++n)
          LoadToLds(to + M::kBytes + n * kWaves * 1024, depth_of(N(), n, kRunsN) < left ? off_n[n] : kNothing, rsrc_n);
      }
    };
    // Steps are on their way to LDS up to kStages ahead. (Past the last
    // zeros, to where nobody reads any more: the number of loads on their way is then always the same.)
    //
    // The two halves of a step's depth take turns: while the matrix cores have one, the fragments of the
    // other come out of LDS. In the middle of a step every wave has all of its fragments in registers
    // and waits for the loads of the next one and for the other waves: from there on the
    // next step can be read, and this one's LDS be loaded into again.
    constexpr int kLoads = M::kLoads + N::kLoads;
    if (steps > 0) {
      StaticFor<kStages>([&](auto d) __attribute__((always_inline)) { issue(d, d); });
      WaitVmcnt<(kStages - 1) * kLoads>();
      Barrier();
      Fragments first, second;
      read(0, 0, first);
      const auto step = [&](int s, auto stage) __attribute__((always_inline)) {
        read(stage, 1, second);
        multiply(first);
        interleave();
        WaitVmcnt<(kStages - 2) * kLoads>();
        Barrier();
        issue(s + kStages, stage);
        read((stage + 1) % kStages, 0, first);
        multiply(second);
        interleave();
      };
      for (int s = 0;;) {
        step(s, std::integral_constant<int, 0>());
        if (++s == steps) break;
        step(s, std::integral_constant<int, 1>());
        if (++s == steps) break;
        if constexpr (kStages > 2) {
          step(s, std::integral_constant<int, 2>());
          if (++s == steps) break;
        }
        if constexpr (kStages > 3) {
          step(s, std::integral_constant<int, 3>());
          if (++s == steps) break;
        }
      }
      // (LDS may be another workgroup's once this one has ended.)
      WaitVmcnt<0>();
    }
  } else {
    // A granule is read where it lies, or, where it would reach past the end of its
    // run, from the run's last 16 bytes (a run has as many); Put then moves it to its place and
    // zeroes what lies past the depth. (What lies past the tile's sides
    // ends up in rows of the tile that are not stored.)
    // Where load n of a lane is in its run and how long the run is, in bytes; `row`, `k`: where the
    // tile begins in the operand. kFar: from step s on (256 bytes are as good as all that is left); addresses of runs along the
    // depth then begin with the step, or, as the run may end less than 16 bytes behind that, 16 bytes in front of it. (Addresses
    // that move with the step cost 2 to 3 % where products are large: 4 x 4095x2047 by 8191, transposed, 217 us and 224.)
    struct Place {
      int at, length;
    };
    constexpr int kBefore = kFar ? 16 : 0;
    const auto place_of = [&](auto side, int n, const Side& from, Runs runs, int row, int s) __attribute__((always_inline)) -> Place {
      using T = decltype(side);
      const int granule = T::GranuleOf(n, wave, lane);
      if (kFar && runs == Runs::kPlain)
        return {granule * 16, min(p.depth - (columns ? 0 : range.begin) - s * E::kDepth, 256 / E::kBytes) * E::kBytes};
      if (runs == Runs::kPlain) return {((columns ? 0 : range.begin) + s * E::kDepth + granule * E::kGranule) * E::kBytes, p.depth * E::kBytes};
      return {(row + granule * E::kGranule) * E::kBytes, from.count * E::kBytes};
    };
    const int row_m = m0, row_n = n0 + (columns ? range.begin : 0);
    // A lane's offsets, from an address that is the same for all: of the run (kPlain) or of the
    // place in it, and of the other of the two, which ends at the operand's end and so goes by the step.
    uint32_t off_m[M::kLoads], off_n[N::kLoads];
    const auto offset_of = [&](auto side, int n, const Side& from, Runs runs, int row, int here) __attribute__((always_inline)) -> uint32_t {
      using T = decltype(side);
      if (runs == Runs::kPlain) return static_cast<uint32_t>(min(T::RunOf(n, wave, lane), here - 1) * from.pitch * E::kBytes);
      const Place where = place_of(side, n, from, runs, row, 0);
      return static_cast<uint32_t>(min(where.at, where.length - 16));
    };
#pragma unroll
    for (int n = 0; n < M::kLoads; ++n) off_m[n] = offset_of(M(), n, p.m, kRunsM, row_m, here_m);
#pragma unroll
    for (int n = 0; n < N::kLoads; ++n) off_n[n] = offset_of(N(), n, p.n, kRunsN, row_n, here_n);
    const auto load_side = [&](auto side, v4i* held, const uint32_t* off, const Side& from, Runs runs, bool dealt_rows, int row,
                               int s) __attribute__((always_inline)) {
      using T = decltype(side);
      const int64_t group = columns && !dealt_rows ? tile.group * from.group_stride : 0;
      const int64_t k = (columns ? 0 : range.begin) + int64_t(s) * E::kDepth;
      const char* const base = static_cast<const char*>(from.data) +
                               (group + (runs == Runs::kPlain ? row : k) * from.pitch) * E::kBytes +
                               (kFar && runs == Runs::kPlain ? k * E::kBytes - kBefore : 0);
      // (Steps have 64 runs at most.)
      const uint32_t last_run = static_cast<uint32_t>(min(depth - 1 - s * E::kDepth, 64) * from.pitch * E::kBytes);
#pragma unroll
      for (int n = 0; n < T::kLoads; ++n) {
        uint32_t other;
        if (runs == Runs::kPlain) {
          const Place where = place_of(side, n, from, runs, row, s);
          other = min(where.at + kBefore, where.length - 16 + kBefore);
        } else {
          other = min(static_cast<uint32_t>(T::RunOf(n, wave, lane) * from.pitch * E::kBytes), last_run);
        }
        held[n] = *reinterpret_cast<const granule::v4i_unaligned*>(base + (off[n] + other));
      }
    };
    // Steps held in registers on their way.
    struct Set {
      v4i m[M::kLoads], n[N::kLoads];
    };
    Set held[2];
    const auto fetch = [&](int s, Set& set) __attribute__((always_inline)) {
      load_side(M(), set.m, off_m, p.m, kRunsM, false, row_m, s);
      load_side(N(), set.n, off_n, p.n, kRunsN, true, row_n, s);
    };
    const auto put_side = [&](auto side, v4i* held, const Side& from, Runs runs, int row, int s, char* to) __attribute__((always_inline)) {
      using T = decltype(side);
      const int k0 = s * E::kDepth;
      const bool depth_ends = k0 + E::kDepth > depth;
      const bool run_ends = runs == Runs::kAcross && int64_t(row) + T::kRows > from.count;
      // (Both the same for the whole workgroup.)
      if (depth_ends || run_ends) {
#pragma unroll
        for (int n = 0; n < T::kLoads; ++n) {
          const Place where = place_of(side, n, from, runs, row, s);
          v4i x = granule::PlaceGranule(held[n], where.at, where.length);
          const int run = T::RunOf(n, wave, lane), granule = T::GranuleOf(n, wave, lane);
          const int left = runs == Runs::kPlain ? depth - k0 - granule * E::kGranule : depth - k0 - run;  // values, or runs
          const int bytes = runs == Runs::kPlain ? left * E::kBytes : left > 0 ? 16 : 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] &= static_cast<int>(granule::LowBytes(bytes - 4 * e));
          held[n] = x;
        }
      }
#pragma unroll
      for (int n = 0; n < T::kLoads; ++n) *reinterpret_cast<v4i*>(to + n * kWaves * 1024) = held[n];
    };
    const auto put = [&](int s, int stage, Set& set) __attribute__((always_inline)) {
      char* to = lds + stage * kStage + (wave * 64 + lane) * 16;
      put_side(M(), set.m, p.m, kRunsM, row_m, s, to);
      put_side(N(), set.n, p.n, kRunsN, row_n, s, to + M::kBytes);
    };
    const auto use = [&](int stage) __attribute__((always_inline)) {
      __syncthreads();
      Fragments first, second;
      read(stage, 0, first);
      read(stage, 1, second);
      multiply(first);
      multiply(second);
    };
    if (steps == 1) {
      fetch(0, held[0]);
      put(0, 0, held[0]);
      use(0);
    } else if (steps > 1) {
      // (Loads past the last step are the last one's again and go unused: the number of loads on
      // their way is then always the same.)
      fetch(0, held[0]);
      fetch(1, held[1]);
      put(0, 0, held[0]);
      fetch(min(2, steps - 1), held[0]);
      const auto next = [&](int s, auto stage) __attribute__((always_inline)) {
        put(s, stage, held[stage]);
        fetch(min(s + 2, steps - 1), held[stage]);
      };
      for (int s = 1;; ++s) {
        use(0);
        if (s == steps) break;
        next(s, std::integral_constant<int, 1>());
        use(1);
        if (++s == steps) break;
        next(s, std::integral_constant<int, 0>());
      }
    }
  }

  // Write-back. Lane l holds column l % 16 of each block of the N side and 4
  // rows (l / 16) * 4 .. of each block of the M side; blocks go in pairs, 8 rows one after the other
  // to a lane. (Those of 16 bits of unpermuted blocks are exchanged between neighbouring rows of 16 lanes for
  // that.) A store takes any address its type allows.
  const int l = lane & 15, q = lane >> 4;
  const bool f32 = p.dst_f32 != 0;
  const int64_t group_at = columns ? 0 : tile.group * p.dst_group_stride;
  const int first_n = columns ? range.begin + n0 : n0;
  const float* bias = p.bias ? p.bias + tile.group * p.bias_stride + m0 : nullptr;
  constexpr bool kPermuted = kRunsM == Runs::kPlain;
  typedef __attribute__((aligned(2))) v4i v4i_of_2;
  typedef __attribute__((aligned(4))) v4f v4f_of_4;
  const auto store = [&](int m, int64_t column, float v) __attribute__((always_inline)) {
    if (m < here_m) StoreFloat(p.dst, f32 ? RUYAMD_DTYPE_F32 : kType, column + (m0 + m) * p.dst_m_stride, v);
  };
#pragma unroll
  for (int i = 0; i < kBlocksM; i += 2) {
    const int rows[2] = {wave_m * M::kWaveRows + M::RowOf(i, q * 4), wave_m * M::kWaveRows + M::RowOf(i + 1, q * 4)};
    float add[2][4] = {};
    if (bias)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) add[h][e] = rows[h] + e < here_m ? bias[rows[h] + e] : 0.0f;
#pragma unroll
    for (int j = 0; j < kBlocksN; ++j) {
      const int n = wave_n * N::kWaveRows + j * 16 + l;
      const int64_t column = group_at + int64_t(first_n + n) * p.dst_n_stride;
      float v[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[h][e] = Clamp(acc[i + h][j][e] + add[h][e], p.clamp_min, p.clamp_max);
      if (p.dst_m_stride != 1) {
        if (n < here_n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) store(rows[h] + e, column, v[h][e]);
        continue;
      }
      if (f32 || kType == RUYAMD_DTYPE_F32) {
        if (n >= here_n) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (rows[h] + 4 <= here_m)
            *reinterpret_cast<v4f_of_4*>(static_cast<float*>(p.dst) + column + m0 + rows[h]) =
                v4f{v[h][0], v[h][1], v[h][2], v[h][3]};
          else
#pragma unroll
            for (int e = 0; e < 4; ++e) store(rows[h] + e, column, v[h][e]);
        }
        continue;
      }
      if constexpr (kType != RUYAMD_DTYPE_F32) {
        v4i packed;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) packed[2 * h + e] = RoundPair<kType>(v[h][2 * e], v[h][2 * e + 1]);
        int m = rows[0];
        if constexpr (!kPermuted) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const auto both = __builtin_amdgcn_permlane16_swap(packed[e], packed[2 + e], false, false);
            packed[e] = both[0];
            packed[2 + e] = both[1];
          }
          m = wave_m * M::kWaveRows + (i + (q & 1)) * 16 + (q >> 1) * 8;
        }
        if (n >= here_n) continue;
        uint16_t* const to = static_cast<uint16_t*>(p.dst) + column + m0 + m;
        if (m + 8 <= here_m) {
          *reinterpret_cast<v4i_of_2*>(to) = packed;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (m + e < here_m) to[e] = static_cast<uint16_t>(static_cast<uint32_t>(packed[e / 2]) >> (16 * (e & 1)));
        }
      }
    }
  }
}

}  // namespace grouped
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_GROUPED_GEMM_H_
