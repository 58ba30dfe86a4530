// Products of 4-bit values on tiles of 256x128, four waves of 128x64, two workgroups to a CU.
//
// One of a CU's two workgroups multiplies while the other waits for its first loads, or for its results to be taken by memory: that
// is what tiles of 256x256, one to a CU, lose on shallow products; and a product needs three quarters of the bytes that it needs on
// 128x128. For two of them to fit LDS steps are of 64 bytes of every row, 128 values: one instruction's depth. Three steps are
// on their way. A wave reads a step's fragments once all of it has landed, and multiplies as they come.
//
// Scales are in LDS as they lie, 16 bytes of a row to four steps; a lane reads those of its rows and takes its column of the four words.
//
// 5120 x 8192 x 512: 27.0 us (256x256 and 128x128 35.6); 16384 x 8192 x 1024 104 (123 and 144); 8192 x 8192 x 2048 83.6 (80.5 and 90.9); 4096 x 4096
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
constexpr int kScales = kStages * kStage, kLds = kScales + kRows * 16;
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

__global__ __launch_bounds__(64 * kWaves, 2) void MxFp4WideKernel(MulCall c) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave_m = wave & 1, wave_n = wave >> 1;
  TileOf tile;
  Range range;
  if (!FindTile(c.offsets, c.groups, c.n, kTileN, (c.m + kTileM - 1) / kTileM, &tile, &range)) return;
  const int m0 = tile.m * kTileM, n0 = tile.n * kTileN;
  const int here_m = min(kTileM, c.m - m0), here_n = min(kTileN, range.count - n0);
  const int steps = c.k / 128, row_scales = c.k / kBlock;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  // The loads: 16 rows each. (Rows past the tile's sides are the last one: they end up in rows of the tile that are not stored.)
  const v4i rsrc_m = Resource(reinterpret_cast<const char*>(c.lhs.data) + tile.group * c.lhs.matrix_bytes + m0 * c.lhs.row_bytes);
  const v4i rsrc_n = Resource(reinterpret_cast<const char*>(c.rhs.data) + (int64_t(range.begin) + n0) * c.rhs.row_bytes);
  uint32_t off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const bool is_m = i < kLoadsM;
    const int r = ((is_m ? i : i - kLoadsM) * kWaves + wave) * 16 + (lane >> 2);
    off[i] = is_m ? static_cast<uint32_t>(min(r, here_m - 1) * c.lhs.row_bytes) + ((lane & 3) ^ Key<true>(r)) * 16
                  : static_cast<uint32_t>(min(r, here_n - 1) * c.rhs.row_bytes) + ((lane & 3) ^ Key<false>(r)) * 16;
  }
  const auto load = [&](auto number, int s, uint32_t stage_at) __attribute__((always_inline)) {
    constexpr int n = decltype(number)::value;
    constexpr int kTo = n < kLoadsM ? n * kWaves * 1024 : kTileM * kRowBytes + (n - kLoadsM) * kWaves * 1024;
    LoadToLds(__builtin_amdgcn_readfirstlane(lds_base + stage_at + wave * 1024 + kTo), off[n], n < kLoadsM ? rsrc_m : rsrc_n,
              __builtin_amdgcn_readfirstlane(s * kRowBytes));
  };
  // Those of scales: 64 rows of the M side to a wave, and 64 of the N side to two waves, and to the other two again.
  const v4i scales_m = Resource(reinterpret_cast<const char*>(c.lhs.scales) + tile.group * c.lhs.scales_matrix_stride + m0 * c.lhs.scale_stride);
  const v4i scales_n = Resource(reinterpret_cast<const char*>(c.rhs.scales) + (int64_t(range.begin) + n0) * c.rhs.scale_stride);
  const uint32_t scales_off_m = static_cast<uint32_t>(min(wave * 64 + lane, here_m - 1) * c.lhs.scale_stride);
  const uint32_t scales_off_n = static_cast<uint32_t>(min((wave & 1) * 64 + lane, here_n - 1) * c.rhs.scale_stride);
  const auto load_scales = [&](int chunk) __attribute__((always_inline)) {
    // (The last 16 of a row, where there are no 16 more.)
    const uint32_t from = __builtin_amdgcn_readfirstlane(min(chunk * 16, row_scales - 16));
    LoadToLds(__builtin_amdgcn_readfirstlane(lds_base + kScales + wave * 1024), scales_off_m, scales_m, from);
    LoadToLds(__builtin_amdgcn_readfirstlane(lds_base + kScales + (kTileM / 64 + (wave & 1)) * 1024), scales_off_n, scales_n, from);
  };

  const int a_row = wave_m * 128 + (l >> 2) * 8 + (l & 3), b_row = wave_n * 64 + l;
  const uint32_t slot = (q ^ (l >> 2)) << 4;  // (both Keys of these rows are l / 4)
  const char* const a_at = lds + a_row * kRowBytes + slot;
  const char* const b_at = lds + (kTileM + b_row) * kRowBytes + slot;
  const auto offset_of_a = [](int i) { return (i >> 1) * 32 + (i & 1) * 4; };  // rows
  const uint32_t selector = ColumnSelector(q);
  int sa[kBlocksM], sb[kBlocksN];
  const auto read_scales = [&](int chunk) __attribute__((always_inline)) {
    v4i raw[kBlocksM + kBlocksN];
#pragma unroll
    for (int j = 0; j < kBlocksN; ++j) raw[j] = *reinterpret_cast<const v4i*>(lds + kScales + (kTileM + b_row + j * 16) * 16);
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i) raw[kBlocksN + i] = *reinterpret_cast<const v4i*>(lds + kScales + (a_row + offset_of_a(i)) * 16);
    if (chunk * 16 + 16 > row_scales) {
#pragma unroll
      for (int i = 0; i < kBlocksM + kBlocksN; ++i) raw[i] = granule::PlaceGranule(raw[i], chunk * 16, row_scales);
    }
#pragma unroll
    for (int j = 0; j < kBlocksN; ++j) sb[j] = ColumnOf(raw[j], selector);
#pragma unroll
    for (int i = 0; i < kBlocksM; ++i) sa[i] = ColumnOf(raw[kBlocksN + i], selector);
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
    WaitVmcnt<kLoads + (kPart == 2 ? 2 : 0)>();
    Barrier();
    if constexpr (kPart == 0) read_scales(s / 4);
    if constexpr (kPart == 1) load_scales(s / 4 + 1);  // (all waves have read the ones before)
    if (s + 2 == steps) {
#pragma unroll
      for (int n = 0; n < kLoads; ++n) off[n] = kNothing;  // (from here on zeros, to where nobody reads)
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

}  // namespace

hipError_t LaunchWide(hipStream_t stream, const MulCall& call, unsigned blocks) {
  static const hipError_t attribute =
      hipFuncSetAttribute(reinterpret_cast<const void*>(MxFp4WideKernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (attribute != hipSuccess) return attribute;
  hipLaunchKernelGGL(MxFp4WideKernel, dim3(blocks), dim3(64 * kWaves), kLds, stream, call);
  return hipGetLastError();
}

}  // namespace mxfp4
}  // namespace ruyamd
