// A tile of a product of 4-bit values on the matrix cores: the steps of the kernels in mxfp4_gemm.hip, and of the largest tile's
// quarters.
//
// Products, LDS reads and loads stand in the order in which they are issued: behind each product what there is of the
// others, so that neither the matrix core nor the address unit waits for the end of a run of the other's. (Left to the compiler, products
// sank behind the barrier: 2048 x 2048 x 8192 on 128x128, four stages 29.0 -> 25.2 us, two 34.9 -> 29.8.) A step of four stages still
// takes 0.65 us at 2.15 GHz, in which the matrix cores are busy for a third (four waves of 64x64 read every fragment out of LDS twice, and
// wait for each other in every step); loads spread over both halves of a step gained nothing.
#ifndef RUY_AMD_CSRC_KERNELS_MXFP4_TILE_H_
#define RUY_AMD_CSRC_KERNELS_MXFP4_TILE_H_

#include "grouped_gemm.h"
#include "mxfp4_device.h"
#include "mxfp4_write_back.h"

#include <type_traits>

namespace ruyamd {
namespace mxfp4 {

using grouped::Barrier;
using grouped::FindTile;
using grouped::kNothing;
using grouped::Range;
using grouped::Resource;
using grouped::Runs;
using grouped::StaticFor;
using grouped::TileOf;
using grouped::TileSide;
using grouped::WaitVmcnt;

// 16 bytes a lane to LDS, from `soffset` bytes behind its offset.
__device__ __forceinline__ void LoadToLds(uint32_t lds, uint32_t voffset, v4i rsrc, uint32_t soffset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"(lds), "v"(voffset), "s"(rsrc), "s"(soffset)
      : "memory");
}

// 4 bytes a lane.
__device__ __forceinline__ void LoadWordToLds(uint32_t lds, uint32_t voffset, v4i rsrc) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %2, 0 offen lds"
      :
      : "s"(lds), "v"(voffset), "s"(rsrc)
      : "memory");
}

// Scales straight to LDS, 16 bytes of a row at a time, of which it has as many at least; where there are no 16 from `first` on the last
// 16 are read, and put in place when they are read there. A load to LDS begins at a multiple of 4 bytes. kWords: rows that begin anywhere,
// or whose number of scales is no multiple of 4: 16 bytes come as the five words that hold them (no byte outside these is read), four to
// a lane and one to a lane, and are shifted. (Where rows are aligned it costs 4 % of 256x256 tiles' time and 10 of the
// others'. 4096 x 4096 x 4064, whose rows have 127 scales: 41.4 us, on 128x128 with scales through registers 57.)
template <bool kWords>
struct ScaleRows {
  static constexpr int kLoads = kWords ? 2 : 1;
  static constexpr int kBytes = kWords ? 20 : 16;  // in LDS
  v4i rsrc;
  uint32_t at;  // the lane's row, in bytes from the resource's base (a multiple of 4)

  __device__ __forceinline__ ScaleRows(const uint8_t* base, int64_t row_offset)
      : rsrc(Resource(reinterpret_cast<const char*>(base) - (reinterpret_cast<uintptr_t>(base) & 3))),
        at(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base) & 3) + static_cast<uint32_t>(row_offset)) {}
  static __device__ __forceinline__ uint32_t From(int first, int count) { return static_cast<uint32_t>(min(first, count - 16)); }
  __device__ __forceinline__ void Load(uint32_t lds, uint32_t lds_words, int first, int count) const {
    if constexpr (kWords) {
      const uint32_t from = at + From(first, count), whole = from & ~3u;
      LoadToLds(lds, whole, rsrc, 0);
      LoadWordToLds(lds_words, whole + (from & 3 ? 16 : 12), rsrc);
    } else {
      LoadToLds(lds, at, rsrc, __builtin_amdgcn_readfirstlane(From(first, count)));
    }
  }
  // `x` and `fifth` (in LDS) are what Load brought.
  static __device__ __forceinline__ v4i Place(v4i x, int fifth, uint32_t row_at, int first, int count) {
    if constexpr (kWords) {
      const uint32_t low = (row_at + From(first, count)) & 3;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = static_cast<int>(__builtin_amdgcn_alignbyte(e < 3 ? x[e + 1] : fifth, x[e], low));
    }
    return granule::PlaceGranule(x, first, count);
  }
};

constexpr int kStep = 8 * kBlock;  // depth positions to a step: 128 bytes

// kDirect: rows of both sides begin at multiples of 4 bytes, which is what a load to LDS asks of an address, and are whole blocks, so
// that tiles go to LDS without passing through registers. (8192 x 8192 x 8192, rows 4100 bytes apart: 263 us, through registers
// 406; 4096 and 4112 apart 245 and 260.) Otherwise rows are read 16 bytes a lane from wherever they begin: 8192 x 8192 x
// 8192, rows 4097 bytes apart 496 to 580 us from card to card. (Reading the five words that hold 16 bytes and shifting them takes 503, and 8 % longer at
// 4096 x 4096 x 4096.)
// kStages: steps on their way to LDS (kDirect), two or four.
// How scales come to LDS. Through registers, a pair of steps ahead: the waves wait for these loads, and for those of all steps with
// them, in every other step, which with more than two stages would be all that the other stages are for. All of the depth's first. Or, where
// a row has 16 of them, as they lie (ScaleRows, with kWords or without), two pairs ahead: then each thread takes its own row's out of
// LDS, and puts them back transposed.
enum class ScaleLoads { kThroughRegisters, kAllFirst, kAhead, kAheadWords };
template <int kWavesM, int kWavesN, int kBlocksM, int kBlocksN, bool kDirect, int kStages, ScaleLoads kScaleLoads>
__device__ __forceinline__ void MultiplyTile(const MulCall& c, const TileOf& tile, const Range& range, char* lds) {
  constexpr int kWaves = kWavesM * kWavesN;
  constexpr int kTileM = kWavesM * kBlocksM * 16, kTileN = kWavesN * kBlocksN * 16;
  // (How rows lie in LDS, which is a matter of bytes alone.)
  using M = TileSide<RUYAMD_DTYPE_BF16, Runs::kPlain, kTileM, kBlocksM, true, kWaves>;
  using N = TileSide<RUYAMD_DTYPE_BF16, Runs::kPlain, kTileN, kBlocksN, false, kWaves>;
  constexpr int kStage = M::kBytes + N::kBytes;
  constexpr bool kAllScales = kScaleLoads == ScaleLoads::kAllFirst;
  constexpr bool kAhead = kScaleLoads == ScaleLoads::kAhead || kScaleLoads == ScaleLoads::kAheadWords;
  using Scaling = ScaleRows<kScaleLoads == ScaleLoads::kAheadWords>;
  constexpr bool kThrough = kScaleLoads == ScaleLoads::kThroughRegisters;
  static_assert(kDirect || (kStages == 2 && kThrough), "");
  constexpr int kRows = kTileM + kTileN, kScalesAt = kStages * kStage, kRawAt = kScalesAt + kRows * 16;
  static_assert(!kAhead || (kRows == 64 * kWaves && kTileM % 64 == 0), "a wave's rows are of one side");
  static_assert(kRows <= 64 * kWaves, "a row's scales to a thread");
  using Out = WriteBack<kBlocksM, kBlocksN>;
  static_assert(kWaves * Out::kLds <= kScalesAt, "");

  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave % kWavesM, wave_n = wave / kWavesM;
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
    *reinterpret_cast<v4i*>(lds + kScalesAt + buffer * (kRows * 16) + row * 16) =
        Transposed(kAhead ? x : PlaceScales(x, pair * 16, row_scales));
  };
  // A thread brings those of one row, pair by pair.
  const uint8_t* const scale_row = scales_of_row(threadIdx.x);
  const auto fetch_scales = [&](int pair) __attribute__((always_inline)) { return LoadScales(scale_row, pair * 16, row_scales); };
  const auto put_scales = [&](const v4i& x, int pair, int buffer) __attribute__((always_inline)) {
    if (kRows == 64 * kWaves || int(threadIdx.x) < kRows) put_scales_of_row(x, threadIdx.x, pair, buffer);
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
    const v4i rsrc_m = Resource(reinterpret_cast<const char*>(base_m)), rsrc_n = Resource(reinterpret_cast<const char*>(base_n));
    constexpr int kLoads = M::kLoads + N::kLoads;
    // What a step that reaches past the depth takes from there are zeros, and all steps behind it.
    const auto end_at = [&](int s) __attribute__((always_inline)) {
      const int left = (c.k - s * kStep) / kBlock;  // granules
      if (left >= 8) return;
#pragma unroll
      for (int n = 0; n < M::kLoads; ++n)
        if (M::GranuleOf(n, wave, lane) >= left) off_m[n] = kNothing;
#pragma unroll
      for (int n = 0; n < N::kLoads; ++n)
        if (N::GranuleOf(n, wave, lane) >= left) off_n[n] = kNothing;
    };
    const auto load = [&](auto number, int s, int stage) __attribute__((always_inline)) {
      constexpr int n = decltype(number)::value;
      const uint32_t to = __builtin_amdgcn_readfirstlane(lds_base + stage * kStage + wave * 1024);
      const uint32_t from = __builtin_amdgcn_readfirstlane(s * 128);
      if constexpr (n < M::kLoads)
        LoadToLds(to + n * kWaves * 1024, off_m[n], rsrc_m, from);
      else
        LoadToLds(to + M::kBytes + (n - M::kLoads) * kWaves * 1024, off_n[n - M::kLoads], rsrc_n, from);
    };
    constexpr int kReads = kBlocksM + kBlocksN, kProducts = kBlocksM * kBlocksN;
    const auto read_one = [&](auto number, int stage, int kk, Fragments& f) __attribute__((always_inline)) {
      constexpr int n = decltype(number)::value;
      const char* const side_m = lds + stage * kStage;
      if constexpr (n < kBlocksN)
        f.n[n] = N::Fragment(side_m + M::kBytes, wave_n, n, kk, lane);
      else
        f.m[n - kBlocksN] = M::Fragment(side_m, wave_m, n - kBlocksN, kk, lane);
    };
    const auto read_scales_one = [&](auto number, int buffer, Scales& s) __attribute__((always_inline)) {
      constexpr int n = decltype(number)::value;
      const char* const at = lds + kScalesAt + buffer * (kRows * 16) + q * 4;
      if constexpr (n < kBlocksN)
        s.n[n] = *reinterpret_cast<const int*>(at + (kTileM + wave_n * N::kWaveRows + N::RowOf(n, l)) * 16);
      else
        s.m[n - kBlocksN] = *reinterpret_cast<const int*>(at + (wave_m * M::kWaveRows + M::RowOf(n - kBlocksN, l)) * 16);
    };
    const auto product = [&](auto number, const Fragments& f, const Scales& s, auto byte) __attribute__((always_inline)) {
      constexpr int i = decltype(number)::value / kBlocksN, j = decltype(number)::value % kBlocksN;
      Mma<decltype(byte)::value>(f.m[i], f.n[j], s.m[i], s.n[j], acc[i][j]);
    };
    // f(i) for those of kAll that come behind product number `at`.
    const auto share = [&](auto at, auto all, auto&& f) __attribute__((always_inline)) {
      constexpr int kFrom = decltype(at)::value * decltype(all)::value / kProducts;
      constexpr int kTo = (decltype(at)::value + 1) * decltype(all)::value / kProducts;
      StaticFor<kTo - kFrom>([&](auto i) __attribute__((always_inline)) { f(std::integral_constant<int, kFrom + decltype(i)::value>()); });
    };
    using Reads = std::integral_constant<int, kReads>;
    using Loads = std::integral_constant<int, kLoads>;
    // As in grouped_gemm.h: steps are on their way to LDS kStages ahead, and the two halves of a step's depth take turns: while the
    // matrix cores have one, the fragments of the other come out of LDS. In the middle of a step all waves wait for the loads
    // of the next one and for each other. With two stages, in every other step the scales of the next pair, which have come with
    // these loads, go into LDS before that, and out of it after.
    v4i next_scales = {};
    if constexpr (kThrough) next_scales = fetch_scales(0);
    // (kAhead: two buffers, of pairs in turn.)
    const int my_row = threadIdx.x & ~63;  // the wave's first one
    const Scaling rows(my_row < kTileM ? c.lhs.scales + tile.group * c.lhs.scales_matrix_stride + m0 * c.lhs.scale_stride
                                       : c.rhs.scales + (int64_t(range.begin) + n0) * c.rhs.scale_stride,
                       my_row < kTileM ? min(my_row + lane, here_m - 1) * c.lhs.scale_stride
                                       : min(my_row - kTileM + lane, here_n - 1) * c.rhs.scale_stride);
    constexpr int kRawBytes = kRows * Scaling::kBytes;  // of a buffer: 16 bytes of all rows, and 4 bytes of all rows
    const auto load_raw = [&](int pair) __attribute__((always_inline)) {
      const uint32_t to = lds_base + kRawAt + (pair & 1) * kRawBytes;
      rows.Load(__builtin_amdgcn_readfirstlane(to + wave * 1024), __builtin_amdgcn_readfirstlane(to + kRows * 16 + wave * 256), pair * 16,
                row_scales);
    };
    const auto read_raw = [&](int pair) __attribute__((always_inline)) {
      const char* const from = lds + kRawAt + (pair & 1) * kRawBytes;
      int fifth = 0;
      if constexpr (Scaling::kLoads > 1) fifth = *reinterpret_cast<const int*>(from + kRows * 16 + threadIdx.x * 4);
      return Scaling::Place(*reinterpret_cast<const v4i*>(from + threadIdx.x * 16), fifth, rows.at, pair * 16, row_scales);
    };
    if constexpr (kAhead) {
      load_raw(0);
      load_raw(1);
    }
    StaticFor<kStages>([&](auto d) __attribute__((always_inline)) {
      end_at(d);
      StaticFor<kLoads>([&](auto n) __attribute__((always_inline)) { load(n, d, d); });
    });
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
    } else if constexpr (kThrough) {
      put_scales(next_scales, 0, 0);
    }
    WaitVmcnt<(kStages - 1) * kLoads>();
    if constexpr (kAhead) put_scales(read_raw(0), 0, 0);
    Barrier();
    Fragments first, second;
    Scales scales, later;
    read(0, 0, first);
    read_scales(0, scales);
    // whole: the loads of the step lie inside the depth.
    const auto step = [&](int s, auto stage, auto whole) __attribute__((always_inline)) {
      constexpr int kAt = decltype(stage)::value, kOdd = kAt % 2, kNext = (kAt + 1) % kStages;
      if constexpr (kStages > 2) end_at(s + kStages);
      StaticFor<kProducts>([&](auto p) __attribute__((always_inline)) {
        product(p, first, scales, std::integral_constant<int, 2 * kOdd>());
        share(p, Reads(), [&](auto r) __attribute__((always_inline)) { read_one(r, kAt, 1, second); });
        __builtin_amdgcn_sched_barrier(0);
      });
      // (kAhead: in odd steps with the loads of scales that went out in the last one; in even ones what they hold has come.)
      WaitVmcnt<(kStages - 2) * kLoads + (kAhead && kOdd ? Scaling::kLoads : 0)>();
      if constexpr (kOdd && !kAllScales) put_scales(next_scales, (s + 1) / 2, 0);
      Barrier();
      if constexpr (!kOdd && kThrough) next_scales = fetch_scales(s / 2 + 1);
      if constexpr (!kOdd && kAhead) {
        next_scales = read_raw(s / 2 + 1);
        load_raw(s / 2 + 2);
      }
      if constexpr (kStages == 2 && !decltype(whole)::value) end_at(s + kStages);
      __builtin_amdgcn_sched_barrier(0);
      StaticFor<kProducts>([&](auto p) __attribute__((always_inline)) {
        product(p, second, scales, std::integral_constant<int, 2 * kOdd + 1>());
        share(p, Reads(), [&](auto r) __attribute__((always_inline)) {
          read_one(r, kNext, 0, first);
          // (Past the last pair: the last one again, of which nothing is used.)
          if constexpr (kOdd) read_scales_one(r, kAllScales ? min((s + 1) / 2, (steps - 1) / 2) : 0, later);
        });
        share(p, Loads(), [&](auto n) __attribute__((always_inline)) { load(n, s + kStages, kAt); });
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (kOdd) scales = later;
    };
    int s = 0;
    // (Two loops for two stages of 128x128 only, 2048 x 2048 x 8192 34.0 -> 30.5 us. Those of 64x64 live on four workgroups to a CU, for
    // which both loops together take too many registers, 36 -> 46; with four stages, whose waves wait less and are alone with
    // the code that they fetch, 25.2 -> 25.7.)
    if constexpr (kStages == 2 && kProducts > 4)
      for (const int whole = c.k / kStep; s + 2 * kStages <= whole; s += kStages)
        StaticFor<kStages>([&](auto d) __attribute__((always_inline)) { step(s + d, d, std::true_type()); });
    for (;;) {
      step(s, std::integral_constant<int, 0>(), std::false_type());
      if (++s == steps) break;
      step(s, std::integral_constant<int, 1>(), std::false_type());
      if (++s == steps) break;
      if constexpr (kStages > 2) {
        step(s, std::integral_constant<int, 2>(), std::false_type());
        if (++s == steps) break;
        step(s, std::integral_constant<int, 3>(), std::false_type());
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

}  // namespace mxfp4
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_MXFP4_TILE_H_
