// Products of 4-bit values of a few columns: every weight is read once, by one wave, straight
// into the registers that the matrix instructions take it from.
//
// A workgroup has some blocks of 16 rows of weights and up to 16 * kCols tokens; its waves deal the
// depth out among themselves, 512 positions (256 bytes of every row) at a time, and add up what they
// have through LDS. The tokens are put into LDS first, with zeros behind the depth, so that
// what is read of the weights there does not matter, and their scales transposed
// (mxfp4_device.h); those of the weights are read where they lie, 16 bytes of a row to a chunk.
//
// HBM bounds it: 16384 x 16384 and one token, 143 MB in 27 us, 5.2 TB/s (a launch and the tokens' way into LDS some 3 us of it; a plain read
// reaches 6.5); 64 experts of 2048 x 2048 and 32 tokens, of which 25 experts have some, 56 MB in 13.6. Loads that go past the caches, or three
// and four chunks on their way and not two, gained nothing. Small ones are a launch and one wave's way through its depth: 2048 x 2048, 5.0 us.
#include "grouped_gemm.h"
#include "launch_geometry.h"
#include "mxfp4_device.h"

#include <algorithm>

namespace ruyamd {
namespace mxfp4 {
namespace {

using grouped::Clamp;
using grouped::FindTile;
using grouped::Range;
using grouped::StoreFloat;
using grouped::TileOf;

struct StreamArgs {
  MulCall c;
  int tiles_m;      // workgroups along the rows
  int depth_waves;  // waves that deal out the depth
  int row_waves;    // waves along the rows (a power of two)
  int pitch;        // bytes from a token in LDS to the next
  int scales_at, scale_pitch;  // the tokens' scales in LDS
  int tokens;       // to a workgroup, at most
};

// LDS that a workgroup may take.
constexpr int kMostLds = 156 << 10;
constexpr int kMostWaves = 16;

template <int kCols>
__global__ __launch_bounds__(64 * kMostWaves) void MxFp4StreamKernel(StreamArgs args) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const MulCall& c = args.c;
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row_wave = wave & (args.row_waves - 1), depth_wave = wave >> __builtin_ctz(args.row_waves);
  const int work_rows = 16 * args.row_waves;
  TileOf tile;
  Range range;
  if (!FindTile(c.offsets, c.groups, c.n, args.tokens, args.tiles_m, &tile, &range)) return;
  const int row0 = tile.m * work_rows, token0 = tile.n * args.tokens;
  const int tokens = min(args.tokens, range.count - token0);
  const int chunks = (c.k + kChunk - 1) / kChunk, whole_chunks = c.k / kChunk;
  const int row_bytes = (c.k + 1) / 2, row_scales = (c.k + kBlock - 1) / kBlock;

  // (Rows past the last are the last one again; their results are not stored.)
  const int64_t my_row = min(row0 + row_wave * 16 + l, c.m - 1);
  const uint8_t* const weights = c.lhs.data + tile.group * c.lhs.matrix_bytes + my_row * c.lhs.row_bytes;
  const uint8_t* const scales = c.lhs.scales + tile.group * c.lhs.scales_matrix_stride + my_row * c.lhs.scale_stride;
  struct Held {
    v4i weights[4], scales;
  };
  // (Loads never reach past the end of a row.)
  const auto load = [&](int chunk, Held& h) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h.weights[i] = granule::LoadGranule<false>(weights, chunk * (kChunk / 2) + i * 64 + q * 16, row_bytes);
    h.scales = LoadScales(scales, chunk * 16, row_scales);
  };
  // This wave's chunks are depth_wave + i * depth_waves, `mine` of them. It starts with another one for each block of rows and
  // goes round: rows lie a power of two apart as often as not, and all waves at one depth would be at few of the memory's channels.
  const int mine = (chunks - depth_wave + args.depth_waves - 1) / args.depth_waves;
  const int start = static_cast<int>(uint32_t(tile.m * args.row_waves + row_wave) % uint32_t(mine));
  const auto chunk_of = [&](int i) __attribute__((always_inline)) {
    const int at = i + start;
    return depth_wave + (at < mine ? at : at - mine) * args.depth_waves;
  };
  Held first, second;
  load(chunk_of(0), first);

  // The tokens, and their scales.
  const uint8_t* const token_data = c.rhs.data + (int64_t(range.begin) + token0) * c.rhs.row_bytes;
  const uint8_t* const token_scales = c.rhs.scales + (int64_t(range.begin) + token0) * c.rhs.scale_stride;
  const uint32_t granules = chunks * 16;
  for (uint32_t i = threadIdx.x; i < tokens * granules; i += blockDim.x) {
    const uint32_t token = i / granules, g = i - token * granules;
    v4i x = granule::LoadGranule<false>(token_data + token * c.rhs.row_bytes, g * 16, row_bytes);
    x = granule::PlaceGranule(x, g * 16, row_bytes);
    *reinterpret_cast<v4i*>(lds + token * args.pitch + g * 16) = WithoutOddHalf(x, int64_t(g) * kBlock, c.k);
  }
  for (uint32_t i = threadIdx.x; i < uint32_t(tokens * chunks); i += blockDim.x) {
    const uint32_t token = i / chunks, chunk = i - token * chunks;
    const v4i x = LoadScales(token_scales + token * c.rhs.scale_stride, chunk * 16, row_scales);
    *reinterpret_cast<v4i*>(lds + args.scales_at + token * args.scale_pitch + chunk * 16) =
        Transposed(PlaceScales(x, chunk * 16, row_scales));
  }
  __syncthreads();

  // Where this lane's tokens are in LDS.
  int token_at[kCols], token_scales_at[kCols];
#pragma unroll
  for (int t = 0; t < kCols; ++t) {
    const int token = min(t * 16 + l, tokens - 1);
    token_at[t] = token * args.pitch + q * 16;
    token_scales_at[t] = args.scales_at + token * args.scale_pitch + q * 4;
  }
  const uint32_t selector = ColumnSelector(q);
  v4f acc[kCols] = {};
  const auto use = [&](int chunk, Held& h) __attribute__((always_inline)) {
    if (chunk >= whole_chunks) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        h.weights[i] = granule::PlaceGranule(h.weights[i], chunk * (kChunk / 2) + i * 64 + q * 16, row_bytes);
      h.scales = PlaceScales(h.scales, chunk * 16, row_scales);
    }
    const int weight_scales = ColumnOf(h.scales, selector);
#pragma unroll
    for (int t = 0; t < kCols; ++t) {
      const char* const x = lds + token_at[t] + chunk * (kChunk / 2);
      const int x_scales = *reinterpret_cast<const int*>(lds + token_scales_at[t] + chunk * 16);
      Mma<0>(h.weights[0], *reinterpret_cast<const v4i*>(x), weight_scales, x_scales, acc[t]);
      Mma<1>(h.weights[1], *reinterpret_cast<const v4i*>(x + 64), weight_scales, x_scales, acc[t]);
      Mma<2>(h.weights[2], *reinterpret_cast<const v4i*>(x + 128), weight_scales, x_scales, acc[t]);
      Mma<3>(h.weights[3], *reinterpret_cast<const v4i*>(x + 192), weight_scales, x_scales, acc[t]);
    }
  };
  // Two chunks of the weights are on their way.
  if (mine > 1) load(chunk_of(1), second);
  for (int i = 0; i < mine; i += 2) {
    use(chunk_of(i), first);
    if (i + 2 < mine) load(chunk_of(i + 2), first);
    if (i + 1 >= mine) break;
    use(chunk_of(i + 1), second);
    if (i + 3 < mine) load(chunk_of(i + 3), second);
  }

  // The waves' sums, added up in the order of the depth, and the write-back. Lane l holds rows
  // (l / 16) * 4 .. of a block for token l % 16.
  float* const partial = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int t = 0; t < kCols; ++t) {
    if (t * 16 >= tokens) break;  // (the same for all waves)
    __syncthreads();
    *reinterpret_cast<v4f*>(partial + wave * 256 + l * 16 + q * 4) = acc[t];
    __syncthreads();
    // Value number v: row v % 16 of a block of 16, block, token.
    for (int v = threadIdx.x; v < work_rows * 16; v += blockDim.x) {
      const int row = v % 16, r = v / 16 & (args.row_waves - 1), token = v / work_rows;
      const int m = row0 + r * 16 + row, n = token0 + t * 16 + token;
      if (m >= c.m || n >= token0 + tokens) continue;
      float sum = 0;
      for (int i = 0; i < args.depth_waves; ++i) sum += partial[(i * args.row_waves + r) * 256 + token * 16 + row];
      if (c.bias) sum += c.bias[tile.group * c.bias_stride + m];
      StoreFloat(c.dst, c.dst_type, m * c.dst_rs + (int64_t(range.begin) + n) * c.dst_cs, Clamp(sum, c.clamp_min, c.clamp_max));
    }
  }
}

template <int kCols>
hipError_t Launch(hipStream_t stream, const StreamArgs& args, unsigned blocks, int waves, unsigned lds) {
  auto* const kernel = &MxFp4StreamKernel<kCols>;
  static const hipError_t attribute =
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
  if (attribute != hipSuccess) return attribute;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * waves), lds, stream, args);
  return hipGetLastError();
}

}  // namespace

bool LaunchStream(hipStream_t stream, const MulCall& call, hipError_t* status) {
  if (call.k < kBlock) return false;  // (a row has 16 bytes at least)
  const bool forced = call.forced_tile_rows == 16 && call.forced_tile_cols == 16;
  if (call.forced_tile_rows && !forced) return false;
  const int64_t busy = std::min(call.groups, call.n);
  // (More than a workgroup has tokens, or, as groups are mostly of many sizes, more than the largest of these would have, who then read
  // their weights again: 64 experts of 2048 x 2048, us here and on tiles: 32 tokens 14.9 and 14.7, 256 35.5 and 32.0; of 4096 x 4096, 16
  // 25.5 and 22.9, 256 134 and 107.)
  if (!forced && call.n > (busy > 1 ? 2 : 32) * busy) return false;
  if (call.k > 0x7fffffff - 2 * kChunk || call.m > 0x7fffffff - 512) return false;
  StreamArgs args;
  args.c = call;
  const int64_t chunks = (int64_t(call.k) + kChunk - 1) / kChunk;
  // (16 tokens side by side, 16 bytes, or a word of scales, of each: all banks once.)
  const int64_t pitch = chunks * (kChunk / 2) + 16, scale_pitch = (chunks * 16 + 255) / 256 * 256 + 16;
  const int64_t fit = kMostLds / (pitch + scale_pitch);
  if (fit < 1) return false;
  const int cols = call.n > 16 * busy && fit > 16 ? 2 : 1;
  args.tokens = static_cast<int>(std::min<int64_t>({16 * cols, fit, call.n}));
  // Waves along the depth: neighbours of a workgroup are at neighbouring chunks, 2 KB of a row with eight. Fewer where they would have less
  // than four chunks each and there are rows for 16 waves to a CU without. (us, one token, eight and four of them: 16384 x 16384
  // 28.0 and 28.3, with two 38; 28672 x 8192 30.1 and 24.8; 2048 x 8192 6.6 and 7.1; 64 experts of 2048 x 2048, 32 tokens, four and
  // one 18.6 and 15.4.) Along the rows as many as make all workgroups fit the CUs, whose LDS the tokens fill, at once, in exchange for
  // waves along the depth where need be. (16 tokens, 16384 x 16384: 8 x 1 65, 8 x 2 39, 4 x 4 35; 32, 8192 x 8192: 8 x 1 29, 8 x 2 16;
  // one, 2048 x 2048: 4 x 1 4.6, 4 x 2 6.0.)
  const int64_t units = (int64_t(call.m) + 15) / 16 * busy;
  int depth_waves = 8, row_waves = 1;
  while (depth_waves > 1 && chunks < 4 * depth_waves && units * depth_waves > int64_t(16) * call.compute_units) depth_waves /= 2;
  while (depth_waves > 1 && chunks < depth_waves) depth_waves /= 2;
  const int64_t tokens_lds = args.tokens * (pitch + scale_pitch), at_once = kMostLds / tokens_lds * call.compute_units;
  while (row_waves < kMostWaves && units > at_once * row_waves) {
    row_waves *= 2;
    if (depth_waves * row_waves > kMostWaves) depth_waves /= 2;
  }
  // About how long this takes, us: a launch, the weights at the rate of a stream, once to each lot of tokens, and a CU's workgroups putting
  // their tokens into LDS. Tiles of many columns read the weights more slowly and go through no more of them for more tokens. Choosing
  // by both costs 1.4 % over the faster one, in the mean over 432 calls of 1 to 256 tokens and weights of 1 to 570 MB. (us, this and the
  // fastest tiles: 16384 x 8192, one token 14.7 and 15.6, 8 18.8 and 15.6, 32 21.7 and 16.0; 2048 x 2048, 16 5.6 and 6.1, 32 7.5 and 6.1;
  // 8 experts of 2048 x 8192, 4 tokens 9.4 and 12.0.)
  const int64_t lots = (call.n + busy * args.tokens - 1) / (busy * args.tokens);
  const double weights = double(busy) * lots * call.m * (call.lhs.row_bytes + call.lhs.scale_stride);
  const int64_t mean_tokens = std::min<int64_t>(args.tokens, (call.n + busy - 1) / busy);
  const int64_t each_cu = (units * lots + int64_t(row_waves) * call.compute_units - 1) / (int64_t(row_waves) * call.compute_units);
  const float time = 4.5f + static_cast<float>(weights / (busy == 1 ? 7.0e6 : 6.0e6)) + 4.5e-5f * float(each_cu * mean_tokens * (pitch + scale_pitch));
  const float tiles = TilesMicroseconds(call);
  if (!forced && tiles >= 0 && tiles < time) return false;
  args.depth_waves = depth_waves;
  args.row_waves = row_waves;
  const int work_rows = 16 * row_waves, waves = depth_waves * row_waves;
  args.tiles_m = (call.m + work_rows - 1) / work_rows;
  args.pitch = static_cast<int>(pitch);
  args.scale_pitch = static_cast<int>(scale_pitch);
  args.scales_at = static_cast<int>(args.tokens * pitch);
  const int64_t lds = std::max(tokens_lds, int64_t(waves) * 1024);
  const int64_t slots = call.n / args.tokens + busy;
  const int64_t blocks = (slots * args.tiles_m + 7) / 8 * 8;
  if (!LaunchFits(blocks, 64 * waves)) return false;
  *status = cols == 2 ? Launch<2>(stream, args, static_cast<unsigned>(blocks), waves, static_cast<unsigned>(lds))
                      : Launch<1>(stream, args, static_cast<unsigned>(blocks), waves, static_cast<unsigned>(lds));
  return true;
}

}  // namespace mxfp4
}  // namespace ruyamd
