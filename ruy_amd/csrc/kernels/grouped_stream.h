// Grouped products of a few columns a group, and products with 4-bit weights:
// every weight is read once, by one workgroup, straight into the registers that
// the matrix instructions take it from.
//
// The 16 columns of a matrix instruction's right-hand side are 16 rows of weights:
// lane l holds the row l % 16, for it 16 bytes at a place that goes by l / 16. The 16
// rows of its left-hand side are tokens; the accumulator of lane l then belongs to
// the weights' row l % 16 and to tokens (l / 16) * 4 .., so that whatever goes with a
// row of weights (a scale, a zero point) is one value to a lane. A workgroup has some
// rows of weights and up to 16 * kCols tokens; its waves deal the depth out among
// themselves, 128 bytes of every row (64 of 4-bit ones) at a time, and add up what they
// have through LDS. The tokens are put into LDS first, as the matrix instructions want
// them: all of their depth where that fits, slab by slab otherwise (kSlabs).
//
// 4-bit weights. (16 + q) is what is left of a 16-bit float of exponent 4 with the four bits of q
// put at the top of its mantissa, so eight of them take eight instructions. Half: 16 + zero is
// then taken away, exactly (packed, half an instruction a weight). bfloat16 has no such
// instruction: the product is formed with 16 + q, and (16 + zero) * sum(x), whose sums come from
// the matrix cores as well (a product with ones), is taken away from every group's sum. fp32 tokens
// are three bf16 rows each that add up to them (float_parts.h), so that every product is exact.
// The scale multiplies a group's sum. Values that are not finite would make 16 + q and 16 + zero
// meet as infinity - infinity; a wave that ends with one goes through its depth once more
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
  int tiles_m;       // workgroups along the rows
  int depth_waves;   // waves that deal out the depth
  int pitch;         // bytes from a token in LDS to the next
  int slab_bytes;    // of one of the two buffers (kSlabs)
};

// LDS that a workgroup of these kernels may take.
constexpr int kStreamLds = 144 << 10;

// How weights of each kind and their tokens come.
template <bool kInt4, int kType>
struct Stream {
  static constexpr int kBytes = kType == RUYAMD_DTYPE_F32 ? 4 : 2;
  static constexpr int kChunk = kInt4 ? 128 : 128 / kBytes;  // depth positions that a wave takes at a time
  static constexpr int kWeightLoads = kInt4 ? 1 : 2;         // of 16 bytes to a row and chunk
  static constexpr int kSteps = kInt4 ? 4 : 2;               // products of a fragment of 16 bytes of tokens
  static constexpr bool kParts = kInt4 && kType == RUYAMD_DTYPE_F32;
  static constexpr int kTokens = kParts ? 5 : 16;            // to 16 rows of a matrix instruction
  static constexpr int kUnit = kInt4 ? 8 : 16 / kBytes;      // depth positions put into LDS at a time
  static constexpr int kUnitLoads = kParts ? 2 : 1;          // of 16 bytes
  static constexpr int kChunkUnits = kChunk / kUnit;         // (16 bytes each in LDS)
};

typedef uint32_t u32_unaligned __attribute__((aligned(1)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef v2i v2i_unaligned __attribute__((aligned(1)));

// Groups of 4-bit weights, by their size: 128 and its multiples, or one for a whole
// row (kWide); 64; 32; any other multiple of 32.
enum class Scaling { kWide, k64, k32, kAny };

// Waves along the rows of a workgroup.
constexpr int RowWaves(bool slabs, int cols) { return slabs && cols > 1 ? 2 : 1; }

template <bool kInt4, int kType, int kRows, int kCols, Scaling kScaling, bool kSlabs>
__global__ __launch_bounds__(512) void GroupedStreamKernel(StreamArgs args) {
  using T = Stream<kInt4, kType>;
  constexpr int kWorkTokens = T::kTokens * kCols;
  constexpr int kRowWaves = RowWaves(kSlabs, kCols);
  constexpr int kWorkRows = 16 * kRows * kRowWaves;
  constexpr int kDepth = 2;  // chunks of weights held by a wave
  // Scales to a chunk, steps to a scale.
  constexpr int kScales = !kInt4 || kScaling == Scaling::kWide ? 1 : kScaling == Scaling::k64 ? 2 : 4;
  constexpr int kStepsToScale = T::kSteps / kScales;
  constexpr bool kScalesSideBySide = kScaling == Scaling::k64 || kScaling == Scaling::k32;
  constexpr bool kHalf = kType == RUYAMD_DTYPE_F16;
  constexpr int kMmaType = kHalf ? RUYAMD_DTYPE_F16 : RUYAMD_DTYPE_BF16;  // of 4-bit weights
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Call& c = args.c;
  const Int4& w = args.w;
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int depth_waves = args.depth_waves;
  const int depth_wave = kRowWaves == 1 ? wave : wave / kRowWaves, row_wave = kRowWaves == 1 ? 0 : wave % kRowWaves;

  TileOf tile;
  Range range;
  if (c.offsets) {
    if (!FindTile<kWorkTokens>(c.offsets, c.groups, c.n, args.tiles_m, &tile, &range)) return;
  } else {
    const int tiles_n = (c.n + kWorkTokens - 1) / kWorkTokens;
    const int64_t all = int64_t(tiles_n) * args.tiles_m, per_xcd = (all + 7) / 8, place = blockIdx.x >> 3;
    const int64_t t = int64_t(blockIdx.x & 7) * per_xcd + place;
    if (place >= per_xcd || t >= all) return;
    tile = {0, static_cast<int>(t / tiles_n), static_cast<int>(t % tiles_n)};
    range = {0, c.n};
  }
  const int row0 = tile.m * kWorkRows, token0 = tile.n * kWorkTokens;
  const int tokens = min(kWorkTokens, range.count - token0);
  const int chunks = (c.k + T::kChunk - 1) / T::kChunk;

  // Where this lane's rows of weights begin. (Rows past the last are the last one
  // again; their results are not stored.)
  const uint8_t* row_data[kRows];
  int64_t row_scales[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = min(row0 + (row_wave * kRows + r) * 16 + l, c.m - 1);
    if constexpr (kInt4) {
      row_data[r] = w.data + tile.group * w.matrix_bytes + row * w.row_bytes;
      row_scales[r] = tile.group * w.scales_matrix_stride + row * w.scale_stride;
    } else {
      row_data[r] = static_cast<const uint8_t*>(c.lhs) + (tile.group * c.matrix_stride + row * c.lhs_rs) * T::kBytes;
    }
  }
  const int row_bytes = kInt4 ? (c.k + 1) / 2 : c.k * T::kBytes;
  const int row_scale_count = kInt4 ? (c.k + w.group_size - 1) / w.group_size : 0;
  const bool f32_scales = w.scale_type == RUYAMD_DTYPE_F32;

  struct Held {
    v4i weights[kRows][T::kWeightLoads];
    uint32_t scales[kRows][kScales], zeros[kRows][kScalesSideBySide ? 1 : kScales];
  };
  // Loads never reach past the end of a row (which has 16 bytes and, side by side,
  // kScales scales at least): what would is read from its last bytes, and moved to
  // where it belongs by Place.
  const auto load = [&](int chunk, Held& h) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < T::kWeightLoads; ++i) {
      const int at = min(chunk * (T::kWeightLoads * 64) + i * 64 + q * 16, row_bytes - 16);
#pragma unroll
      for (int r = 0; r < kRows; ++r) h.weights[r][i] = *reinterpret_cast<const granule::v4i_unaligned*>(row_data[r] + at);
    }
    if constexpr (kInt4) {
      if constexpr (kScalesSideBySide) {
        const int at = min(chunk * kScales, row_scale_count - kScales);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          if (f32_scales) {
            const float* p = static_cast<const float*>(w.scales) + row_scales[r] + at;
#pragma unroll
            for (int g = 0; g < kScales; ++g) h.scales[r][g] = __float_as_uint(p[g]);
          } else {
            const uint16_t* p = static_cast<const uint16_t*>(w.scales) + row_scales[r] + at;
            if constexpr (kScales == 4) {
              const v2i both = *reinterpret_cast<const v2i_unaligned*>(p);
              h.scales[r][0] = both[0];
              h.scales[r][1] = both[1];
            } else {
              h.scales[r][0] = *reinterpret_cast<const u32_unaligned*>(p);
            }
          }
          h.zeros[r][0] = 0x08080808u;
          if (w.zero_points) {
            const uint8_t* p = w.zero_points + row_scales[r] + at;
            h.zeros[r][0] = kScales == 4 ? *reinterpret_cast<const u32_unaligned*>(p) : p[0] | p[1] << 8;
          }
        }
      } else {
#pragma unroll
        for (int g = 0; g < kScales; ++g) {
          const int at = w.group_size == 128 ? chunk : min(chunk * 128 + g * 32, c.k - 1) / w.group_size;
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            h.scales[r][g] = f32_scales ? static_cast<const uint32_t*>(w.scales)[row_scales[r] + at]
                                        : static_cast<const uint16_t*>(w.scales)[row_scales[r] + at];
            h.zeros[r][g] = w.zero_points ? w.zero_points[row_scales[r] + at] : 8;
          }
        }
      }
    }
  };
  const auto place = [&](int chunk, Held& h) __attribute__((always_inline)) {
    if ((chunk + 1) * T::kChunk <= c.k) return;
#pragma unroll
    for (int i = 0; i < T::kWeightLoads; ++i) {
      const int at = chunk * (T::kWeightLoads * 64) + i * 64 + q * 16;
#pragma unroll
      for (int r = 0; r < kRows; ++r) h.weights[r][i] = granule::PlaceGranule(h.weights[r][i], at, row_bytes);
    }
    if constexpr (kInt4 && kScalesSideBySide) {
      for (int past = (chunk + 1) * kScales - row_scale_count; past > 0; --past)
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          h.zeros[r][0] >>= 8;
          if (f32_scales) {
#pragma unroll
            for (int g = 0; g < kScales; ++g) h.scales[r][g] = g + 1 < kScales ? h.scales[r][g + 1] : 0;
          } else {
            h.scales[r][0] >>= 16;
            if constexpr (kScales == 4) {
              h.scales[r][0] |= h.scales[r][1] << 16;
              h.scales[r][1] >>= 16;
            }
          }
        }
    }
  };
  const auto scale_of = [&](const Held& h, int r, int g) __attribute__((always_inline)) -> float {
    if (f32_scales) return __uint_as_float(h.scales[r][g]);
    const uint32_t bits = kScalesSideBySide ? h.scales[r][g / 2] >> (16 * (g & 1)) & 0xffffu : h.scales[r][g];
    if (w.scale_type == RUYAMD_DTYPE_BF16) return __uint_as_float(bits << 16);
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
  };
  const auto zero_of = [&](const Held& h, int r, int g) __attribute__((always_inline)) -> uint32_t {
    return kScalesSideBySide ? h.zeros[r][0] >> (8 * g) & 0xffu : h.zeros[r][g];
  };

  // Unit u of a token (kUnit values from depth position u * kUnit on), zeros past the depth.
  struct Unit {
    v4i x[T::kUnitLoads];
  };
  const auto fetch = [&](int token, int u) __attribute__((always_inline)) -> Unit {
    Unit unit;
    const int k = u * T::kUnit;
    const uint8_t* p = static_cast<const uint8_t*>(c.rhs) +
                       ((int64_t(range.begin) + token0 + token) * c.rhs_cs + k * c.rhs_rs) * T::kBytes;
    if (c.rhs_rs == 1 && k + T::kUnit <= c.k) {
#pragma unroll
      for (int i = 0; i < T::kUnitLoads; ++i) unit.x[i] = reinterpret_cast<const granule::v4i_unaligned*>(p)[i];
      return unit;
    }
    // One value after the other, each pushed in behind those before it.
#pragma unroll
    for (int i = 0; i < T::kUnitLoads; ++i) {
      constexpr int kValues = 16 / T::kBytes;
      v4i x = {0, 0, 0, 0};
#pragma unroll 1
      for (int e = 0; e < kValues; ++e) {
        uint32_t v = 0;
        const int at = i * kValues + e;
        if (k + at < c.k) {
          if constexpr (T::kBytes == 4)
            v = *reinterpret_cast<const uint32_t*>(p + at * c.rhs_rs * 4);
          else
            v = *reinterpret_cast<const uint16_t*>(p + at * c.rhs_rs * 2);
        }
        if constexpr (T::kBytes == 4) {
          x = v4i{x[1], x[2], x[3], static_cast<int>(v)};
        } else {
          x = v4i{static_cast<int>(__builtin_amdgcn_alignbyte(x[1], x[0], 2)),
                  static_cast<int>(__builtin_amdgcn_alignbyte(x[2], x[1], 2)),
                  static_cast<int>(__builtin_amdgcn_alignbyte(x[3], x[2], 2)),
                  static_cast<int>(__builtin_amdgcn_alignbyte(v, x[3], 2))};
        }
      }
      unit.x[i] = x;
    }
    return unit;
  };
  // 8 values of 16 bits in the order 0 4 1 5 2 6 3 7, in which 4-bit values come out of a word.
  const auto in_word_order = [&](v4i x) __attribute__((always_inline)) -> v4i {
    return v4i{static_cast<int>(__builtin_amdgcn_perm(x[2], x[0], 0x05040100)),
               static_cast<int>(__builtin_amdgcn_perm(x[2], x[0], 0x07060302)),
               static_cast<int>(__builtin_amdgcn_perm(x[3], x[1], 0x05040100)),
               static_cast<int>(__builtin_amdgcn_perm(x[3], x[1], 0x07060302))};
  };
  // `to`: the unit's place in its token's first row of LDS.
  const auto put = [&](const Unit& unit, char* to) __attribute__((always_inline)) {
    if constexpr (!kInt4) {
      *reinterpret_cast<v4i*>(to) = unit.x[0];
    } else if constexpr (!T::kParts) {
      *reinterpret_cast<v4i*>(to) = in_word_order(unit.x[0]);
    } else {
      v4i high, middle, low;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = __int_as_float(unit.x[0][e]), y = __int_as_float(unit.x[1][e]);
        high[e] = float_parts::RoundPair(x, y);
        x -= float_parts::LowHalf(high[e]);
        y -= float_parts::HighHalf(high[e]);
        middle[e] = float_parts::RoundPair(x, y);
        x -= float_parts::LowHalf(middle[e]);
        y -= float_parts::HighHalf(middle[e]);
        low[e] = float_parts::RoundPair(x, y);
      }
      *reinterpret_cast<v4i*>(to) = high;
      *reinterpret_cast<v4i*>(to + args.pitch) = middle;
      *reinterpret_cast<v4i*>(to + 2 * args.pitch) = low;
    }
  };
  const auto row_in_lds = [&](int token) __attribute__((always_inline)) -> int {
    return T::kParts ? token / 5 * 16 + token % 5 * 3 : token;
  };
  // Row of LDS that this lane reads of 16 rows of tokens (one that holds a token).
  int lds_row[kCols];
#pragma unroll
  for (int t = 0; t < kCols; ++t) {
    const int here = max(1, min(T::kTokens, tokens - t * T::kTokens)) * (T::kParts ? 3 : 1);
    lds_row[t] = (t * T::kTokens < tokens ? t * 16 : 0) + min(l, here - 1);
  }

  v4f acc[kRows][kCols] = {};

  // 16 + q of the eight values of a word, in that order.
  const auto sixteen_and = [&](uint32_t x) __attribute__((always_inline)) -> v4i {
    constexpr uint32_t kSixteen = kHalf ? 0x4C004C00u : 0x41804180u, kMask = kHalf ? 0x03C003C0u : 0x00780078u;
    constexpr int kUp = kHalf ? 6 : 3;
    v4i out;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int shift = kUp - 4 * e;
      out[e] = static_cast<int>(((shift >= 0 ? x << (shift & 31) : x >> (-shift & 31)) & kMask) | kSixteen);
    }
    return out;
  };
  // 16-byte pieces of four lanes to pieces of a 4-byte word each: word j of the
  // lane with q holds what bytes j * 16 + q * 4 .. of the row's 64 held. A step's 32 depth positions are
  // then consecutive, as scales to fewer than 128 need it.
  const auto exchange = [&](v4i x) __attribute__((always_inline)) -> v4i {
    if constexpr (kScaling == Scaling::kWide) return x;
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
  // The unit of a chunk that step j of this lane takes.
  const auto unit_of = [&](int j) __attribute__((always_inline)) -> int {
    return kInt4 && kScaling == Scaling::kWide ? q * 4 + j : j * 4 + q;
  };

  // `at`: the chunk's place in the tokens' rows.
  const auto use = [&](const Held& h, const char* at) __attribute__((always_inline)) {
    if constexpr (!kInt4) {
#pragma unroll
      for (int j = 0; j < T::kSteps; ++j)
#pragma unroll
        for (int t = 0; t < kCols; ++t) {
          const v4i x = *reinterpret_cast<const v4i*>(at + lds_row[t] * args.pitch + unit_of(j) * 16);
#pragma unroll
          for (int r = 0; r < kRows; ++r) Mma<kType>(x, h.weights[r][j], acc[r][t]);
        }
    } else {
      v4i words[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) words[r] = exchange(h.weights[r][0]);
#pragma unroll
      for (int g = 0; g < kScales; ++g) {
        v4f sum[kRows][kCols] = {};
        v4f ones[kCols] = {};
#pragma unroll
        for (int f = 0; f < kStepsToScale; ++f) {
          const int j = g * kStepsToScale + f;
          v4i x[kCols];
#pragma unroll
          for (int t = 0; t < kCols; ++t) {
            x[t] = *reinterpret_cast<const v4i*>(at + lds_row[t] * args.pitch + unit_of(j) * 16);
            if constexpr (!kHalf) {
              constexpr int kOnes = 0x3F803F80;
              Mma<kMmaType>(x[t], v4i{kOnes, kOnes, kOnes, kOnes}, ones[t]);
            }
          }
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            v4i b = sixteen_and(words[r][j]);
            if constexpr (kHalf) {
              const auto sixteen_and_zero = static_cast<uint16_t>(0x4C00u | zero_of(h, r, g) << 6);
              b = __builtin_bit_cast(v4i, __builtin_bit_cast(v8h, b) - __builtin_bit_cast(_Float16, sixteen_and_zero));
            }
#pragma unroll
            for (int t = 0; t < kCols; ++t) Mma<kMmaType>(x[t], b, sum[r][t]);
          }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float scale = scale_of(h, r, g);
          const float away = -16.0f - static_cast<float>(zero_of(h, r, g));
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

  Held held[kDepth];
  StaticFor<kDepth>([&](auto d) __attribute__((always_inline)) {
    const int chunk = depth_wave + d * depth_waves;
    if (chunk < chunks) load(chunk, held[d]);
  });
  constexpr int kLdsChunk = T::kChunkUnits * 16;
  const int iterations = (chunks + depth_waves - 1) / depth_waves;
  // Units of a slab that a thread puts into LDS.
  constexpr int kPieces = (kWorkTokens * T::kChunkUnits + 64 * kRowWaves - 1) / (64 * kRowWaves);
  Unit pieces[kSlabs ? kPieces : 1];
  const int slab_units = depth_waves * T::kChunkUnits, unit_bits = __builtin_ctz(slab_units);  // (a power of two)
  const auto fetch_slab = [&](int slab) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int n = i * blockDim.x + threadIdx.x;
      if (n < tokens * slab_units) pieces[i] = fetch(n >> unit_bits, slab * slab_units + (n & (slab_units - 1)));
    }
  };
  const auto put_slab = [&](int buffer) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int n = i * blockDim.x + threadIdx.x;
      if (n < tokens * slab_units)
        put(pieces[i], lds + buffer * args.slab_bytes + row_in_lds(n >> unit_bits) * args.pitch +
                           (n & (slab_units - 1)) * 16);
    }
  };
  if constexpr (kSlabs) {
    fetch_slab(0);
    put_slab(0);
    if (iterations > 1) fetch_slab(1);
  } else {
    const int units = chunks * T::kChunkUnits;
    for (int n0 = threadIdx.x; n0 < tokens * units; n0 += 4 * blockDim.x) {
      Unit some[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = n0 + i * blockDim.x;
        if (n < tokens * units) some[i] = fetch(n / units, n % units);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = n0 + i * blockDim.x;
        if (n < tokens * units) put(some[i], lds + row_in_lds(n / units) * args.pitch + n % units * 16);
      }
    }
    __syncthreads();
  }
  for (int i = 0; i < iterations; i += kDepth) {
    StaticFor<kDepth>([&](auto d) __attribute__((always_inline)) {
      const int n = i + d, chunk = depth_wave + n * depth_waves;
      if (kSlabs && n < iterations) {
        // Slab n is there, and slab n - 1 no longer read, when all have come here.
        __syncthreads();
        if (n + 1 < iterations) put_slab((n + 1) & 1);
        if (n + 2 < iterations) fetch_slab(n + 2);
      }
      if (chunk < chunks) {
        place(chunk, held[d]);
        use(held[d], kSlabs ? lds + (n & 1) * args.slab_bytes + depth_wave * kLdsChunk : lds + chunk * kLdsChunk);
        if (chunk + kDepth * depth_waves < chunks) load(chunk + kDepth * depth_waves, held[d]);
      }
    });
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
      for (int chunk = depth_wave; chunk < chunks; chunk += depth_waves) {
        Held h;
        load(chunk, h);
        place(chunk, h);
#pragma unroll
        for (int r = 0; r < kRows; ++r) h.weights[r][0] = exchange(h.weights[r][0]);
#pragma unroll
        for (int g = 0; g < kScales; ++g) {
#pragma unroll 1
          for (int f = 0; f < kStepsToScale; ++f) {
            const int j = g * kStepsToScale + f;
#pragma unroll
            for (int t = 0; t < kCols; ++t) {
              // (fp32: the whole token in the place of its first part.)
              const int token = min(t * T::kTokens + (T::kParts ? l / 3 : l), tokens - 1);
              const Unit x = fetch(token, chunk * T::kChunkUnits + unit_of(j));
#pragma unroll
              for (int r = 0; r < kRows; ++r) {
                const uint32_t word = h.weights[r][0][0];
                const int zero = static_cast<int>(zero_of(h, r, g));
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(static_cast<int>(word >> (4 * e) & 15) - zero);
                v4f sum = {0, 0, 0, 0};
                if constexpr (T::kParts) {
#pragma unroll
                  for (int e = 0; e < 8; ++e)
                    sum = __builtin_amdgcn_mfma_f32_16x16x4f32(l % 3 == 0 ? __int_as_float(x.x[e / 4][e % 4]) : 0.0f, v[e],
                                                               sum, 0, 0, 0);
                } else {
                  const v4i b = {float_parts::RoundPair(v[0], v[4]), float_parts::RoundPair(v[1], v[5]),
                                 float_parts::RoundPair(v[2], v[6]), float_parts::RoundPair(v[3], v[7])};
                  Mma<kMmaType>(in_word_order(x.x[0]), b, sum);
                }
                const float scale = scale_of(h, r, g);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][t][e] = __builtin_fmaf(scale, sum[e], acc[r][t][e]);
              }
            }
            // (The next step's word in the place of this one's.)
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
              const v4i x = h.weights[r][0];
              h.weights[r][0] = v4i{x[1], x[2], x[3], 0};
            }
          }
        }
      }
    }
  }

  // The waves' sums, added up in the order of the depth, and the write-back.
  float* const partial = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int t = 0; t < kCols; ++t) {
    if (t * T::kTokens >= tokens) break;  // (the same for all waves)
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) partial[((wave * kRows + r) * 4 + e) * 64 + lane] = acc[r][t][e];
    __syncthreads();
    // Value number v: row v % 16 of a block of 16, token v / 16 % 16, block v / 256.
    for (int v = threadIdx.x; v < kWorkRows * T::kTokens; v += blockDim.x) {
      const int row = v % 16, token = v / 16 % T::kTokens, r = v / (16 * T::kTokens);
      const int m = row0 + r * 16 + row, n = token0 + t * T::kTokens + token;
      if (m >= c.m || n >= token0 + tokens) continue;
      float sum = 0;
#pragma unroll
      for (int s = 0; s < (T::kParts ? 3 : 1); ++s) {
        const int at = T::kParts ? token * 3 + s : token;  // row of the accumulators' block
        const float* from = partial + (r * 4 + at % 4) * 64 + at / 4 * 16 + row;
        for (int i = 0; i < depth_waves; ++i) sum += from[i * kRowWaves * kRows * 256];
      }
      if (c.bias) sum += c.bias[tile.group * c.bias_stride + m];
      StoreFloat(c.dst, c.dst_type, m * c.dst_rs + (int64_t(range.begin) + n) * c.dst_cs,
                 Clamp(sum, c.clamp_min, c.clamp_max));
    }
  }
}

// What a launch needs beside its arguments.
struct StreamPlan {
  unsigned blocks;
  int waves;
  int rows, cols;  // kRows and kCols of the kernel
  bool slabs;
  Scaling scaling;
  unsigned lds_bytes;
};

template <bool kInt4, int kType, int kRows, int kCols, Scaling kScaling, bool kSlabs>
hipError_t LaunchStreamKernel(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  auto* const kernel = &GroupedStreamKernel<kInt4, kType, kRows, kCols, kScaling, kSlabs>;
  static const hipError_t attribute = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, kStreamLds);
  if (attribute != hipSuccess) return attribute;
  hipLaunchKernelGGL(kernel, dim3(plan.blocks), dim3(64 * plan.waves), plan.lds_bytes, stream, args);
  return hipGetLastError();
}

template <bool kInt4, int kType, Scaling kScaling, int kRows>
hipError_t LaunchStreamRows(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  if constexpr (kInt4 && kRows == 1) {
    if (plan.cols == 4) return LaunchStreamKernel<kInt4, kType, 1, 4, kScaling, true>(stream, args, plan);
  }
  if constexpr (kRows <= 2) {
    if (plan.cols == 2) return LaunchStreamKernel<kInt4, kType, kRows, 2, kScaling, true>(stream, args, plan);
  }
  if (plan.slabs) return LaunchStreamKernel<kInt4, kType, kRows, 1, kScaling, true>(stream, args, plan);
  return LaunchStreamKernel<kInt4, kType, kRows, 1, kScaling, false>(stream, args, plan);
}

template <bool kInt4, int kType, Scaling kScaling>
hipError_t LaunchStreamScaling(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  if constexpr (!kInt4)
    if (plan.rows == 4) return LaunchStreamRows<kInt4, kType, kScaling, 4>(stream, args, plan);
  if (plan.rows == 2) return LaunchStreamRows<kInt4, kType, kScaling, 2>(stream, args, plan);
  return LaunchStreamRows<kInt4, kType, kScaling, 1>(stream, args, plan);
}

template <int kType>
hipError_t LaunchStreamInt4(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  switch (plan.scaling) {
    case Scaling::kWide:
      return LaunchStreamScaling<true, kType, Scaling::kWide>(stream, args, plan);
    case Scaling::k64:
      return LaunchStreamScaling<true, kType, Scaling::k64>(stream, args, plan);
    case Scaling::k32:
      return LaunchStreamScaling<true, kType, Scaling::k32>(stream, args, plan);
    default:
      return LaunchStreamRows<true, kType, Scaling::kAny, 1>(stream, args, plan);
  }
}

// (Each in a file of its own.)
hipError_t LaunchStreamInt4Bf16(hipStream_t, const StreamArgs&, const StreamPlan&);
hipError_t LaunchStreamInt4F16(hipStream_t, const StreamArgs&, const StreamPlan&);
hipError_t LaunchStreamInt4F32(hipStream_t, const StreamArgs&, const StreamPlan&);

}  // namespace grouped
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_GROUPED_STREAM_H_
