// Grouped products of a few columns a group, and products with 4-bit weights:
// every weight is read once, by one workgroup, straight into the registers that
// the matrix instructions take it from.
//
// The 16 columns of a matrix instruction's right-hand side are 16 rows of weights:
// lane l holds the row l % 16, for it 16 bytes at a place that goes by l / 16. The 16
// rows of its left-hand side are tokens; the accumulator of lane l then belongs to
// the weights' row l % 16 and to tokens (l / 16) * 4 .., so that whatever goes with a
// row of weights (a scale, a zero point) is one value to a lane. A workgroup has 16 * kRows rows of
// weights and up to 16 * kCols tokens; its waves deal the depth out among
// themselves, 128 bytes of every row (64 of 4-bit ones) at a time, and add up what they have through LDS.
//
// 4-bit weights. (16 + q) is what is left of a 16-bit float of exponent 4 with the four bits of q
// put at the top of its mantissa, so eight of them take eight instructions. Half: 16 + zero is
// then taken away, exactly (packed, half an instruction a weight). bfloat16 has no such
// instruction: the product is formed with 16 + q, and (16 + zero) * sum(x), whose sums come from
// the matrix cores as well (a product with ones), is taken away from every group's sum. fp32 tokens
// are three bf16 columns each that add up to them (float_parts.h), so that every product is exact.
// The scale multiplies a group's sum. Values that are not finite would make 16 + q and 16 + zero meet as
// infinity - infinity; a wave that ends with one goes through its depth once more
// with the exact q - zero.
#ifndef RUY_AMD_CSRC_KERNELS_GROUPED_STREAM_H_
#define RUY_AMD_CSRC_KERNELS_GROUPED_STREAM_H_

#include "float_parts.h"
#include "grouped_gemm.h"

namespace ruyamd {
namespace grouped {

struct StreamArgs {
  Call c;
  Int4 w;
  int row_blocks;  // workgroups along the rows
};

typedef unsigned short u16_unaligned __attribute__((aligned(1)));

// How weights of each kind and their tokens come: depth positions to a chunk,
// loads of 16 bytes to a chunk and row.
template <bool kInt4, int kType>
struct Stream {
  static constexpr int kBytes = kType == RUYAMD_DTYPE_F32 ? 4 : 2;
  static constexpr int kChunk = kInt4 ? 128 : 128 / kBytes;
  static constexpr int kWeightLoads = kInt4 ? 1 : 2;
  // Products of 32 depth positions each (16 of fp32 weights).
  static constexpr int kSteps = kInt4 ? 4 : 2;
  static constexpr bool kParts = kInt4 && kType == RUYAMD_DTYPE_F32;
  // Granules of a token to a step.
  static constexpr int kTokenGranules = kParts ? 2 : 1;
  // Tokens to 16 rows of a matrix instruction.
  static constexpr int kTokens = kParts ? 5 : 16;
  static constexpr int kStepDepth = kChunk / kSteps;
};

// A group's sums are scaled after every kFlush steps of 32 depth positions: 4
// (a scale to 128 positions or a multiple) or 1.
template <bool kInt4, int kType, int kRows, int kCols, int kFlush, int kMostWaves>
__global__ __launch_bounds__(64 * kMostWaves) void GroupedStreamKernel(StreamArgs args) {
  using T = Stream<kInt4, kType>;
  constexpr int kWorkTokens = T::kTokens * kCols;
  constexpr int kGroupsPerChunk = kInt4 ? T::kSteps / kFlush : 1;
  const Call& c = args.c;
  const Int4& w = args.w;
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  __shared__ float partial[kMostWaves * kRows * 256];

  TileOf tile;
  Range range;
  if (!FindTile<kWorkTokens>(c.offsets, c.groups, c.n, args.row_blocks, &tile, &range)) return;
  const int row0 = tile.m * 16 * kRows, token0 = tile.n * kWorkTokens;
  const int tokens = min(kWorkTokens, range.count - token0);

  // Where this lane's rows of weights and its tokens begin. (Rows and tokens past
  // the last are the last one again; their results are not stored.)
  const uint8_t* row_data[kRows];
  int64_t row_scales[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = min(row0 + r * 16 + l, c.m - 1);
    if constexpr (kInt4) {
      row_data[r] = w.data + tile.group * w.matrix_bytes + row * w.row_bytes;
      row_scales[r] = tile.group * w.scales_matrix_stride + row * w.scale_stride;
    } else {
      row_data[r] = static_cast<const uint8_t*>(c.lhs) + (tile.group * c.matrix_stride + row * c.lhs_rs) * T::kBytes;
    }
  }
  const uint8_t* token_data[kCols];
#pragma unroll
  for (int t = 0; t < kCols; ++t) {
    const int token = min(token0 + t * T::kTokens + (T::kParts ? l / 3 : l), token0 + tokens - 1);
    token_data[t] = static_cast<const uint8_t*>(c.rhs) + (int64_t(range.begin) + token) * c.rhs_cs * T::kBytes;
  }
  const int part = T::kParts ? l % 3 : 0;
  const int row_bytes = kInt4 ? (c.k + 1) / 2 : c.k * T::kBytes;
  const int last_scale = kInt4 ? (c.k - 1) / w.group_size : 0;

  struct Held {
    v4i weights[kRows][T::kWeightLoads];
    v4i tokens[kCols][T::kSteps][T::kTokenGranules];
    uint32_t scales[kRows][kGroupsPerChunk], zeros[kRows][kGroupsPerChunk];
  };
  const auto load_scales = [&](int k0, Held& h) __attribute__((always_inline)) {
    if constexpr (kInt4) {
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int g = 0; g < kGroupsPerChunk; ++g) {
          const int64_t at = row_scales[r] + min((k0 + g * 32 * kFlush) / w.group_size, last_scale);
          h.scales[r][g] = w.scale_type == RUYAMD_DTYPE_F32 ? static_cast<const uint32_t*>(w.scales)[at]
                                                            : static_cast<const uint16_t*>(w.scales)[at];
          h.zeros[r][g] = w.zero_points ? w.zero_points[at] : 8;
        }
    }
  };

  // Chunks that lie inside the depth, of tokens whose values lie side by side.
  const auto load = [&](int chunk, Held& h) __attribute__((always_inline)) {
    const int k0 = chunk * T::kChunk;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < T::kWeightLoads; ++i)
        h.weights[r][i] = *reinterpret_cast<const granule::v4i_unaligned*>(
            row_data[r] + chunk * (T::kWeightLoads * 64) + i * 64 + q * 16);
    load_scales(k0, h);
#pragma unroll
    for (int t = 0; t < kCols; ++t)
#pragma unroll
      for (int j = 0; j < T::kSteps; ++j)
#pragma unroll
        for (int i = 0; i < T::kTokenGranules; ++i)
          h.tokens[t][j][i] = *reinterpret_cast<const granule::v4i_unaligned*>(
              token_data[t] + (k0 + j * T::kStepDepth) * T::kBytes + (q * T::kTokenGranules + i) * 16);
  };
  // Any chunk, zeros past the depth (of which a row has 16 bytes at least).
  const auto load_any = [&](int chunk, Held& h) __attribute__((always_inline)) {
    const int k0 = chunk * T::kChunk;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < T::kWeightLoads; ++i) {
        const int at = chunk * (T::kWeightLoads * 64) + i * 64 + q * 16;
        h.weights[r][i] = granule::PlaceGranule(granule::LoadGranule<false>(row_data[r], at, row_bytes), at, row_bytes);
      }
    load_scales(k0, h);
#pragma unroll
    for (int t = 0; t < kCols; ++t)
#pragma unroll
      for (int j = 0; j < T::kSteps; ++j)
#pragma unroll
        for (int i = 0; i < T::kTokenGranules; ++i) {
          const int at = (k0 + j * T::kStepDepth) * T::kBytes + (q * T::kTokenGranules + i) * 16;
          if (c.rhs_rs == 1) {
            h.tokens[t][j][i] = granule::PlaceGranule(granule::LoadGranule<false>(token_data[t], at, c.k * T::kBytes), at,
                                                      c.k * T::kBytes);
          } else {
            v4i x = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 16 / T::kBytes; ++e) {
              const int k = at / T::kBytes + e;
              if (k >= c.k) continue;
              const uint8_t* p = token_data[t] + k * c.rhs_rs * T::kBytes;
              if constexpr (T::kBytes == 4)
                x[e] = *reinterpret_cast<const int*>(p);
              else
                x[e / 2] |= static_cast<int>(uint32_t(*reinterpret_cast<const uint16_t*>(p)) << (16 * (e & 1)));
            }
            h.tokens[t][j][i] = x;
          }
        }
  };

  v4f acc[kRows][kCols] = {};

  // Half and bfloat16 tokens: the 8 values of a granule in the order 0 4 1 5 2 6 3 7, in
  // which 4-bit values come out of a word. fp32 tokens: this lane's part of them.
  const auto token_operand = [&](const v4i (&g)[T::kTokenGranules]) __attribute__((always_inline)) -> v4i {
    if constexpr (!kInt4) {
      return g[0];
    } else if constexpr (!T::kParts) {
      const v4i x = g[0];
      return v4i{static_cast<int>(__builtin_amdgcn_perm(x[2], x[0], 0x05040100)),
                 static_cast<int>(__builtin_amdgcn_perm(x[2], x[0], 0x07060302)),
                 static_cast<int>(__builtin_amdgcn_perm(x[3], x[1], 0x05040100)),
                 static_cast<int>(__builtin_amdgcn_perm(x[3], x[1], 0x07060302))};
    } else {
      v4i out;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = __int_as_float(g[0][e]), y = __int_as_float(g[1][e]);
        const int high = float_parts::RoundPair(x, y);
        x -= float_parts::LowHalf(high);
        y -= float_parts::HighHalf(high);
        const int middle = float_parts::RoundPair(x, y);
        x -= float_parts::LowHalf(middle);
        y -= float_parts::HighHalf(middle);
        const int low = float_parts::RoundPair(x, y);
        out[e] = part == 0 ? high : part == 1 ? middle : low;
      }
      return out;
    }
  };
  const auto scale_of = [&](uint32_t bits) __attribute__((always_inline)) -> float {
    if (w.scale_type == RUYAMD_DTYPE_F32) return __uint_as_float(bits);
    if (w.scale_type == RUYAMD_DTYPE_BF16) return __uint_as_float(bits << 16);
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
  };
  constexpr bool kHalf = kType == RUYAMD_DTYPE_F16;
  constexpr int kMmaType = kHalf ? RUYAMD_DTYPE_F16 : RUYAMD_DTYPE_BF16;  // of 4-bit weights
  // 16 + q of the eight values of a word, in that order.
  const auto sixteen_and = [&](uint32_t x) __attribute__((always_inline)) -> v4i {
    constexpr uint32_t kOne = kHalf ? 0x4C004C00u : 0x41804180u, kMask = kHalf ? 0x03C003C0u : 0x00780078u;
    constexpr int kUp = kHalf ? 6 : 3;
    v4i out;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int shift = kUp - 4 * e;
      out[e] = static_cast<int>(((shift >= 0 ? x << (shift & 31) : x >> (-shift & 31)) & kMask) | kOne);
    }
    return out;
  };
  // 16-byte pieces of four lanes to pieces of a 4-byte word each: word j of the
  // lane with q holds what bytes j * 16 + q * 4 .. of the row's 64 held.
  const auto exchange = [&](v4i x) __attribute__((always_inline)) -> v4i {
    // (Words 0, 1 of the upper half of the lanes against words 2, 3 of the lower one, then odd
    // rows of 16 lanes against even ones.)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const auto p = __builtin_amdgcn_permlane32_swap(x[e], x[e + 2], false, false);
      x[e] = p[0];
      x[e + 2] = p[1];
    }
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const auto p = __builtin_amdgcn_permlane16_swap(x[e], x[e + 1], false, false);
      x[e] = p[0];
      x[e + 1] = p[1];
    }
    return x;
  };

  const auto use = [&](const Held& h) __attribute__((always_inline)) {
    if constexpr (!kInt4) {
#pragma unroll
      for (int j = 0; j < T::kSteps; ++j)
#pragma unroll
        for (int t = 0; t < kCols; ++t)
#pragma unroll
          for (int r = 0; r < kRows; ++r) Mma<kType>(h.tokens[t][j][0], h.weights[r][j], acc[r][t]);
    } else {
      v4i words[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) words[r] = exchange(h.weights[r][0]);
#pragma unroll
      for (int g = 0; g < kGroupsPerChunk; ++g) {
        v4f sum[kRows][kCols] = {};
        v4f ones[kCols] = {};
#pragma unroll
        for (int f = 0; f < kFlush; ++f) {
          const int j = g * kFlush + f;
          v4i x[kCols];
#pragma unroll
          for (int t = 0; t < kCols; ++t) {
            x[t] = token_operand(h.tokens[t][j]);
            if constexpr (!kHalf) {
              constexpr int kOnes = 0x3F803F80;
              Mma<kMmaType>(x[t], v4i{kOnes, kOnes, kOnes, kOnes}, ones[t]);
            }
          }
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            v4i b = sixteen_and(words[r][j]);
            if constexpr (kHalf) {
              const auto sixteen_and_zero = static_cast<uint16_t>(0x4C00u | h.zeros[r][g] << 6);
              b = __builtin_bit_cast(v4i, __builtin_bit_cast(v8h, b) - __builtin_bit_cast(_Float16, sixteen_and_zero));
            }
#pragma unroll
            for (int t = 0; t < kCols; ++t) Mma<kMmaType>(x[t], b, sum[r][t]);
          }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float scale = scale_of(h.scales[r][g]);
          const float away = -16.0f - static_cast<float>(h.zeros[r][g]);
#pragma unroll
          for (int t = 0; t < kCols; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = sum[r][t][e];
              if constexpr (!kHalf) v = __builtin_fmaf(away, ones[t][e], v);
              acc[r][t][e] = __builtin_fmaf(scale, v, acc[r][t][e]);
            }
        }
      }
    }
  };

  const int chunks = (c.k + T::kChunk - 1) / T::kChunk;
  const int plain_chunks = c.rhs_rs == 1 ? c.k / T::kChunk : 0;
  int chunk = wave;
  {
    Held a, b;
    if (chunk < plain_chunks) load(chunk, a);
    while (chunk < plain_chunks) {
      if (chunk + waves < plain_chunks) load(chunk + waves, b);
      use(a);
      chunk += waves;
      if (chunk >= plain_chunks) break;
      if (chunk + waves < plain_chunks) load(chunk + waves, a);
      use(b);
      chunk += waves;
    }
  }
#pragma unroll 1
  for (; chunk < chunks; chunk += waves) {
    Held h;
    load_any(chunk, h);
    use(h);
  }

  if constexpr (kInt4 && !kHalf) {
    bool finite = true;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int t = 0; t < kCols; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) finite = finite && __builtin_isfinite(acc[r][t][e]);
    if (__any(!finite)) {
      // Once more, with q - zero itself: exact in bfloat16 and in fp32.
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int t = 0; t < kCols; ++t) acc[r][t] = v4f{0, 0, 0, 0};
#pragma unroll 1
      for (int again = wave; again < chunks; again += waves) {
        Held h;
        load_any(again, h);
#pragma unroll
        for (int r = 0; r < kRows; ++r) h.weights[r][0] = exchange(h.weights[r][0]);
        // (One step's code: the next step's words, tokens and scales are moved to its place.)
#pragma unroll 1
        for (int j = 0; j < T::kSteps; ++j) {
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const float scale = scale_of(h.scales[r][0]);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              v[e] = static_cast<float>((h.weights[r][0][0] >> (4 * e) & 15) - static_cast<int>(h.zeros[r][0]));
#pragma unroll
            for (int t = 0; t < kCols; ++t) {
              v4f sum = {0, 0, 0, 0};
              if constexpr (T::kParts) {
                // The whole token in the place of its first part.
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  sum = __builtin_amdgcn_mfma_f32_16x16x4f32(
                      part == 0 ? __int_as_float(h.tokens[t][0][e / 4][e % 4]) : 0.0f, v[e], sum, 0, 0, 0);
              } else {
                const v4i b = {float_parts::RoundPair(v[0], v[4]), float_parts::RoundPair(v[1], v[5]),
                               float_parts::RoundPair(v[2], v[6]), float_parts::RoundPair(v[3], v[7])};
                Mma<kMmaType>(token_operand(h.tokens[t][0]), b, sum);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[r][t][e] = __builtin_fmaf(scale, sum[e], acc[r][t][e]);
            }
            const v4i words = h.weights[r][0];
            h.weights[r][0] = v4i{words[1], words[2], words[3], 0};
#pragma unroll
            for (int g = 0; g + 1 < kGroupsPerChunk; ++g) {
              h.scales[r][g] = h.scales[r][g + 1];
              h.zeros[r][g] = h.zeros[r][g + 1];
            }
          }
#pragma unroll
          for (int t = 0; t < kCols; ++t)
#pragma unroll
            for (int s = 0; s + 1 < T::kSteps; ++s)
#pragma unroll
              for (int i = 0; i < T::kTokenGranules; ++i) h.tokens[t][s][i] = h.tokens[t][s + 1][i];
        }
      }
    }
  }

  // The waves' sums, added up in the order of the waves, and the write-back.
#pragma unroll
  for (int t = 0; t < kCols; ++t) {
    if (t > 0) __syncthreads();
    if (t * T::kTokens >= tokens) break;  // (the same for all waves)
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) partial[((wave * kRows + r) * 4 + e) * 64 + lane] = acc[r][t][e];
    __syncthreads();
    // Value number v: row v % 16 of a block of 16, token v / 16 % 16, block v / 256.
    for (int v = threadIdx.x; v < kRows * 16 * T::kTokens; v += blockDim.x) {
      const int row = v % 16, token = v / 16 % T::kTokens, r = v / (16 * T::kTokens);
      const int m = row0 + r * 16 + row, n = token0 + t * T::kTokens + token;
      float sum = 0;
#pragma unroll
      for (int s = 0; s < (T::kParts ? 3 : 1); ++s) {
        const int at = T::kParts ? token * 3 + s : token;  // row of the accumulators' block
        const float* from = partial + (r * 4 + at % 4) * 64 + at / 4 * 16 + row;
        for (int i = 0; i < waves; ++i) sum += from[i * kRows * 256];
      }
      if (m < c.m && n < token0 + tokens) {
        if (c.bias) sum += c.bias[tile.group * c.bias_stride + m];
        StoreFloat(c.dst, c.dst_type, m * c.dst_rs + (int64_t(range.begin) + n) * c.dst_cs,
                   Clamp(sum, c.clamp_min, c.clamp_max));
      }
    }
  }
}

// One launch; kInt4 and kType are fixed, the rest goes by `rows` (of 16, to a
// workgroup) and `cols` (of 16 or 5 tokens).
template <bool kInt4, int kType, int kRows, int kCols>
void LaunchStreamOf(hipStream_t stream, const StreamArgs& args, unsigned blocks, int waves) {
  constexpr int kMostWaves = 8;
  const dim3 grid(blocks), block(64 * waves);
  if constexpr (!kInt4) {
    hipLaunchKernelGGL((GroupedStreamKernel<false, kType, kRows, kCols, 1, kMostWaves>), grid, block, 0, stream, args);
  } else if (args.w.group_size % 128 == 0 || args.w.group_size >= args.c.k) {
    hipLaunchKernelGGL((GroupedStreamKernel<true, kType, kRows, kCols, 4, kMostWaves>), grid, block, 0, stream, args);
  } else {
    hipLaunchKernelGGL((GroupedStreamKernel<true, kType, kRows, kCols, 1, kMostWaves>), grid, block, 0, stream, args);
  }
}

template <bool kInt4, int kType>
hipError_t LaunchStreamType(hipStream_t stream, const StreamArgs& args, unsigned blocks, int waves, int rows, int cols) {
  const auto with_cols = [&](auto kr) {
    constexpr int kRows = decltype(kr)::value;
    if (cols == 1) return LaunchStreamOf<kInt4, kType, kRows, 1>(stream, args, blocks, waves);
    if (cols == 2) return LaunchStreamOf<kInt4, kType, kRows, 2>(stream, args, blocks, waves);
    if constexpr (kInt4) LaunchStreamOf<kInt4, kType, kRows, 4>(stream, args, blocks, waves);
  };
  if (rows == 1)
    with_cols(std::integral_constant<int, 1>());
  else if (rows == 2)
    with_cols(std::integral_constant<int, 2>());
  else
    with_cols(std::integral_constant<int, 4>());
  return hipGetLastError();
}

// (Each in a file of its own.)
hipError_t LaunchStreamInt4Bf16(hipStream_t, const StreamArgs&, unsigned blocks, int waves, int rows, int cols);
hipError_t LaunchStreamInt4F16(hipStream_t, const StreamArgs&, unsigned blocks, int waves, int rows, int cols);
hipError_t LaunchStreamInt4F32(hipStream_t, const StreamArgs&, unsigned blocks, int waves, int rows, int cols);

}  // namespace grouped
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_GROUPED_STREAM_H_
