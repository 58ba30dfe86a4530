// Products of 4-bit values on tiles of 256x128, four waves of 128x64, two workgroups to a CU.
//
// One of a CU's two workgroups multiplies while the other waits for its first loads, or for its results to be taken by memory: that
// is what tiles of 256x256, one to a CU, lose on shallow products; and a product needs three quarters of the bytes that it needs on
// 128x128. For two of them to fit LDS steps are of 64 bytes of every row, 128 values: one instruction's depth. Three steps are
// on their way. A wave reads a step's fragments once all of it has landed, and multiplies as they come.
//
// Scales are in LDS as they lie, 16 bytes of a row to four steps; a lane reads those of its rows and takes its column of the four words.
//
// 5120 x 8192 x 512: 27.3 us (256x256 34.2, 128x128 33.2); 16384 x 8192 x 1024 104 to 115 (118 to 123 and 134 to 144; three calls in turn, whose
// destinations of 268 MB no cache holds, 132 to 137); 8192 x 8192 x 2048 83.6 (80.5 and 90.9); 4096 x 4096
// x 32768, where nothing but the steps counts, 296 (207 and 290). Its loads, of half a line of 16 rows each, take a CU longer than those of a line of
// 8: without them the last one is 231.
#include "mxfp4_large.h"
#include "mxfp4_tile.h"

namespace ruyamd {
namespace mxfp4 {
namespace {

constexpr int kTileM = 256, kTileN = 128, kRows = kTileM + kTileN, kWaves = 4;
constexpr int kBlocksM = 8, kBlocksN = 4;
constexpr int kRowBytes = 64, kStages = 3, kStage = kRows * kRowBytes;
constexpr int kScales = kStages * kStage, kFifths = kScales + kRows * 16, kLds = kFifths + kRows * 4;
constexpr int kLoadsM = kTileM * kRowBytes / 1024 / kWaves, kLoadsN = kTileN * kRowBytes / 1024 / kWaves, kLoads = kLoadsM + kLoadsN;
using Out = WriteBack<kBlocksM, kBlocksN>;
static_assert(kWaves * Out::kLds <= kLds, "");
static_assert(2 * kLds <= 160 << 10, "two workgroups to a CU");

// Granule g of row r lies in slot g ^ Key(r) of its step: the 16 rows that are read together, and of them four to 256 bytes, then
// are in all of these. On the M side they are as in TileSide (8 consecutive rows to two blocks).
template <bool kM>
__device__ __forceinline__ int Key(int r) {
  return kM ? (r >> 3) & 3 : (r >> 2) & 3;
}

template <bool kWords>
__global__ __launch_bounds__(64 * kWaves, 2) void MxFp4WideKernel(MulCall c) {
  using Scaling = ScaleRows<kWords>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave_m = wave & 1, wave_n = wave >> 1;
  TileOf tile;
  Range range;
  if (!FindTile(c.offsets, c.groups, c.n, kTileN, (c.m + kTileM - 1) / kTileM, &tile, &range)) return;
  const int m0 = tile.m * kTileM, n0 = tile.n * kTileN;
  const int here_m = min(kTileM, c.m - m0), here_n = min(kTileN, range.count - n0);
  const int steps = (c.k + 127) / 128, row_scales = c.k / kBlock;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  // The loads: 16 rows each. (Rows past the tile's sides are the last one: they end up in rows of the tile that are not stored.)
  const v4i rsrc_m = Resource(reinterpret_cast<const char*>(c.lhs.data) + tile.group * c.lhs.matrix_bytes + m0 * c.lhs.row_bytes);
  const v4i rsrc_n = Resource(reinterpret_cast<const char*>(c.rhs.data) + (int64_t(range.begin) + n0) * c.rhs.row_bytes);
  uint32_t off[kLoads];
  const auto row_of = [&](int n, int of_lane) __attribute__((always_inline)) {
    return ((n < kLoadsM ? n : n - kLoadsM) * kWaves + wave) * 16 + (of_lane >> 2);
  };
  const auto granule_of = [&](int n, int of_lane) __attribute__((always_inline)) {
    return (of_lane & 3) ^ (n < kLoadsM ? Key<true>(row_of(n, of_lane)) : Key<false>(row_of(n, of_lane)));
  };
#pragma unroll
  for (int n = 0; n < kLoads; ++n)
    off[n] = static_cast<uint32_t>(n < kLoadsM ? min(row_of(n, lane), here_m - 1) * c.lhs.row_bytes : min(row_of(n, lane), here_n - 1) * c.rhs.row_bytes) +
             granule_of(n, lane) * 16;
  const auto load = [&](auto number, int s, uint32_t stage_at) __attribute__((always_inline)) {
    constexpr int n = decltype(number)::value;
    constexpr int kTo = n < kLoadsM ? n * kWaves * 1024 : kTileM * kRowBytes + (n - kLoadsM) * kWaves * 1024;
    LoadToLds(__builtin_amdgcn_readfirstlane(lds_base + stage_at + wave * 1024 + kTo), off[n], n < kLoadsM ? rsrc_m : rsrc_n,
              __builtin_amdgcn_readfirstlane(s * kRowBytes));
  };
  // Those of scales: 64 rows of the M side to a wave, and 64 of the N side to two waves, and to the other two again.
  const uint8_t* const scales_m = c.lhs.scales + tile.group * c.lhs.scales_matrix_stride + m0 * c.lhs.scale_stride;
  const uint8_t* const scales_n = c.rhs.scales + (int64_t(range.begin) + n0) * c.rhs.scale_stride;
  const Scaling rows_m(scales_m, min(wave * 64 + lane, here_m - 1) * c.lhs.scale_stride);
  const Scaling rows_n(scales_n, min((wave & 1) * 64 + lane, here_n - 1) * c.rhs.scale_stride);
  const auto load_scales = [&](int chunk) __attribute__((always_inline)) {
    const int n = kTileM / 64 + (wave & 1);
    rows_m.Load(__builtin_amdgcn_readfirstlane(lds_base + kScales + wave * 1024), __builtin_amdgcn_readfirstlane(lds_base + kFifths + wave * 256),
                chunk * 16, row_scales);
    rows_n.Load(__builtin_amdgcn_readfirstlane(lds_base + kScales + n * 1024), __builtin_amdgcn_readfirstlane(lds_base + kFifths + n * 256),
                chunk * 16, row_scales);
  };

  const int a_row = wave_m * 128 + (l >> 2) * 8 + (l & 3), b_row = wave_n * 64 + l;
  const uint32_t slot = (q ^ (l >> 2)) << 4;  // (both Keys of these rows are l / 4)
  const char* const a_at = lds + a_row * kRowBytes + slot;
  const char* const b_at = lds + (kTileM + b_row) * kRowBytes + slot;
  const auto offset_of_a = [](int i) { return (i >> 1) * 32 + (i & 1) * 4; };  // rows
  int sa[kBlocksM], sb[kBlocksN];
  // What is needed once to four steps, or at the end, is made of the lane's number then: registers are few.
  const auto lane_again = [&]() __attribute__((always_inline)) {
    int v = threadIdx.x;
    asm volatile("" : "+v"(v));
    return v & 63;
  };
  const auto read_scales = [&](int chunk) __attribute__((always_inline)) {
    const int lane2 = lane_again(), l2 = lane2 & 15;
    const int a_row2 = wave_m * 128 + (l2 >> 2) * 8 + (l2 & 3), b_row2 = wave_n * 64 + l2;
    const uint32_t selector = ColumnSelector(lane2 >> 4);
    // (A lane's rows of a side are multiples of 4 apart: what is left of their addresses by 4 is the same.)
    const uint32_t a_low = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(scales_m)) + static_cast<uint32_t>(a_row2) * static_cast<uint32_t>(c.lhs.scale_stride);
    const uint32_t b_low = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(scales_n)) + static_cast<uint32_t>(b_row2) * static_cast<uint32_t>(c.rhs.scale_stride);
    const auto column = [&](int row, uint32_t low) __attribute__((always_inline)) {
      int fifth = 0;
      if constexpr (kWords) fifth = *reinterpret_cast<const int*>(lds + kFifths + row * 4);
      const v4i x = *reinterpret_cast<const v4i*>(lds + kScales + row * 16);
      return ColumnOf(Scaling::Place(x, fifth, low, chunk * 16, row_scales), selector);
    };
#pragma unroll
    for (int j = 0; j < kBlocksN; ++j) sb[j] = column(kTileM + b_row2 + j * 16, b_low);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i) {
      sa[i] = column(a_row2 + offset_of_a(i), a_low);
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  };

  v4f acc[kBlocksM][kBlocksN] = {};
  load_scales(0);
  StaticFor<2>([&](auto d) __attribute__((always_inline)) {
    StaticFor<kLoads>([&](auto n) __attribute__((always_inline)) { load(n, d, d * kStage); });
  });
  uint32_t at = 0, free_at = 2 * kStage;  // the step's stage, and that of the step before it, which the one two steps on gets
  // Step s, number `part` of the four that a chunk of scales has. Its loads have landed when those of the next step, and what went
  // out with them, are all that is left.
  const auto step = [&](int s, auto part) __attribute__((always_inline)) {
    constexpr int kPart = decltype(part)::value;
    WaitVmcnt<kLoads + (kPart == 2 ? 2 * Scaling::kLoads : 0)>();
    Barrier();
    if constexpr (kPart == 0) read_scales(s / 4);
    if constexpr (kPart == 1) load_scales(s / 4 + 1);  // (all waves have read the ones before)
    const int left = row_scales - (s + 2) * 4;  // granules of the step that is loaded
    if (left < 4) {
      const int of_lane = lane_again();
#pragma unroll
      for (int n = 0; n < kLoads; ++n)
        if (granule_of(n, of_lane) >= left) off[n] = kNothing;  // (zeros past the depth, from here on)
    }
    v4i a[kBlocksM], b[kBlocksN];
#pragma unroll
    for (int j = 0; j < kBlocksN; ++j) b[j] = *reinterpret_cast<const v4i*>(b_at + at + j * 16 * kRowBytes);
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i) a[i] = *reinterpret_cast<const v4i*>(a_at + at + offset_of_a(i) * kRowBytes);
    __builtin_amdgcn_sched_barrier(0);
    StaticFor<kBlocksM>([&](auto i) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) Mma<kPart>(a[i], b[j], sa[i], sb[j], acc[i][j]);
      if constexpr (decltype(i)::value < kLoads) load(i, s + 2, free_at);
      __builtin_amdgcn_sched_barrier(0);
    });
    free_at = at;
    at = at == (kStages - 1) * kStage ? 0 : at + kStage;
  };
  for (int s = 0;;) {
    step(s, std::integral_constant<int, 0>());
    if (++s == steps) break;
    step(s, std::integral_constant<int, 1>());
    if (++s == steps) break;
    step(s, std::integral_constant<int, 2>());
    if (++s == steps) break;
    step(s, std::integral_constant<int, 3>());
    if (++s == steps) break;
  }
  WaitVmcnt<0>();

  // (LDS is the write-back's now.)
  __syncthreads();
  const int row0 = wave_m * 128, column0 = wave_n * 64;
  Out{c, acc, lds + wave * Out::kLds, c.bias ? c.bias + tile.group * c.bias_stride + m0 + row0 : nullptr, m0 + row0,
      int64_t(range.begin) + n0 + column0, here_m - row0, here_n - column0}();
}

template <bool kWords>
hipError_t Launch(hipStream_t stream, const MulCall& call, unsigned blocks) {
  static const hipError_t attribute =
      hipFuncSetAttribute(reinterpret_cast<const void*>(&MxFp4WideKernel<kWords>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (attribute != hipSuccess) return attribute;
  hipLaunchKernelGGL(MxFp4WideKernel<kWords>, dim3(blocks), dim3(64 * kWaves), kLds, stream, call);
  return hipGetLastError();
}

}  // namespace

hipError_t LaunchWide(hipStream_t stream, const MulCall& call, unsigned blocks) {
  return ScalesNeedWords(call) ? Launch<true>(stream, call, blocks) : Launch<false>(stream, call, blocks);
}

}  // namespace mxfp4
}  // namespace ruyamd
