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
// 4-bit weights. What is multiplied is q - zero, exactly, whatever the tokens' type: any other
// sum, from which the zero point's share is taken away later, is rounded by values that the
// result does not have, without bound where a large token meets weights equal to their zero
// point. The four bits of q put into the mantissa of 1024 as a half make 1024 + q, two at a
// time. Half: 1024 + zero is then taken away, packed: 9 instructions to 8 weights. bfloat16 has
// no such instruction: 1024 + zero is taken away in fp32, and the upper halves of the results,
// which have all of them, are the bfloat16 values: 17 instructions (64 x 2048x2048 with a scale
// to 32, below, 22.4 us; with products of 16 + q, two at a time, and their sums put right
// afterwards 20.5). fp32 tokens are three bf16 rows each that add up to them (float_parts.h),
// so that every product is exact, against the same weights. The scale multiplies a group's
// sum. Values that are not finite would meet as parts of infinity - infinity, and most below 2^-110 are
// not the sum of their parts, whose remainders show it; a wave that ends with the former, and all waves of
// a workgroup that meets one of the latter, go through their depth once more with whole values.
//
// What bounds it is the rate of the weights' bytes out of HBM. Half, 64 matrices of
// 2048x2048, 25 of them with one of 32 tokens or more: 210 MB in 40.6 us, 5.2 TB/s; 4-bit,
// 16384x16384 with a scale to 128, one token: 138 MB in 30.7 us, 4.5 TB/s (6.5 TB/s is the
// most that anything here reads at). The taking apart of 4-bit values is 0.6 of these and putting the scales into LDS
// 1.9; with a scale to 32 and bfloat16, 64 x 2048x2048, 59 MB in 22.4 us, they are 4.9 and 3.1 (each left out alone, in
// a copy). Small ones are one wave's way through its depth: 2048x2048 5.4 us of which 2.5 are the launch.
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
  int depth_waves;   // waves that deal out the depth (a power of two)
  int row_waves;     // waves along the rows (a power of two; kSlabs: RowWaves)
  int pitch;         // bytes from a token in LDS to the next
  int slab_bytes;    // of one of the two buffers (kSlabs)
  int tokens;        // to a workgroup, at most
  int scale_shift;   // Scaling::kWide: logarithm of the depth positions to a scale
  int scales_at, scale_pitch;  // scales of 4-bit weights in LDS: bytes, values from a row to the next
  int zeros_at, zero_pitch;    // and their zero points
  int lost_at;  // a flag to each wave (fp32 tokens of 4-bit weights)
};

// LDS that a workgroup of these kernels may take.
constexpr int kStreamLds = 156 << 10;

// How weights of each kind and their tokens come. A wave takes 128 bytes of every row
// at a time, a whole line of the caches (4-bit weights slab by slab: 64, half the tokens
// in LDS).
template <bool kInt4, int kType, bool kSlabs>
struct Stream {
  static constexpr int kBytes = kType == RUYAMD_DTYPE_F32 ? 4 : 2;
  static constexpr int kChunk = kInt4 ? (kSlabs ? 128 : 256) : 128 / kBytes;  // depth positions
  static constexpr int kWeightLoads = kInt4 && kSlabs ? 1 : 2;  // of 16 bytes to a row and chunk
  static constexpr int kSteps = (kInt4 ? 4 : 1) * kWeightLoads; // products of a fragment of 16 bytes of tokens
  static constexpr bool kParts = kInt4 && kType == RUYAMD_DTYPE_F32;
  static constexpr int kTokens = kParts ? 5 : 16;            // to 16 rows of a matrix instruction
  static constexpr int kUnit = kInt4 ? 8 : 16 / kBytes;      // depth positions put into LDS at a time
  static constexpr int kUnitLoads = kParts ? 2 : 1;          // of 16 bytes
  static constexpr int kChunkUnits = kChunk / kUnit;         // (16 bytes each in LDS)
};

typedef uint32_t u32_unaligned __attribute__((aligned(1)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef v2i v2i_unaligned __attribute__((aligned(1)));

// Groups of 4-bit weights, by their size: a power of two from 128 on, or one for a whole
// row (kWide); 64; 32; any other multiple of 32.
enum class Scaling { kWide, k64, k32, kAny };

// Waves along the rows of a workgroup of the kernels that go slab by slab.
constexpr int RowWaves(bool slabs, int cols) { return slabs && cols > 1 ? 2 : 1; }

template <bool kInt4, int kType, int kCols, Scaling kScaling, bool kSlabs, bool kZeroPoints>
__global__ __launch_bounds__(512) void GroupedStreamKernel(StreamArgs args) {
  using T = Stream<kInt4, kType, kSlabs>;
  constexpr int kMostTokens = T::kTokens * kCols;
  constexpr int kRowWaves = RowWaves(kSlabs, kCols);
  // Scales to a chunk, steps to a scale.
  constexpr int kScales =
      T::kWeightLoads * (!kInt4 || kScaling == Scaling::kWide ? 1 : kScaling == Scaling::k64 ? 2 : 4);
  constexpr int kStepsToScale = kInt4 ? T::kSteps / kScales : 1;
  constexpr bool kScalesInLds = kInt4 && kScaling != Scaling::kAny;
  constexpr bool kHalf = kType == RUYAMD_DTYPE_F16;
  constexpr int kMmaType = kHalf ? RUYAMD_DTYPE_F16 : RUYAMD_DTYPE_BF16;  // of 4-bit weights
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Call& c = args.c;
  const Int4& w = args.w;
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int depth_waves = args.depth_waves, row_waves = kSlabs ? kRowWaves : args.row_waves;
  const int depth_wave = wave >> __builtin_ctz(row_waves), row_wave = wave & (row_waves - 1);
  const int work_rows = 16 * row_waves;

  TileOf tile;
  Range range;
  if (c.offsets) {
    if (!FindTile(c.offsets, c.groups, c.n, args.tokens, args.tiles_m, &tile, &range)) return;
  } else {
    const int tiles_n = (c.n + args.tokens - 1) / args.tokens;
    const int64_t all = int64_t(tiles_n) * args.tiles_m, per_xcd = (all + 7) / 8, place = blockIdx.x >> 3;
    const int64_t t = int64_t(blockIdx.x & 7) * per_xcd + place;
    if (place >= per_xcd || t >= all) return;
    tile = {0, static_cast<int>(t / tiles_n), static_cast<int>(t % tiles_n)};
    range = {0, c.n};
  }
  const int row0 = tile.m * work_rows, token0 = tile.n * args.tokens;
  const int tokens = min(args.tokens, range.count - token0);
  const int chunks = (c.k + T::kChunk - 1) / T::kChunk, whole_chunks = c.k / T::kChunk;

  // Where this lane's rows of weights begin. (Rows past the last are the last one
  // again; their results are not stored.)
  const uint8_t* row_data;
  int64_t row_scales;
  const int64_t my_row = min(row0 + row_wave * 16 + l, c.m - 1);
  if constexpr (kInt4) {
    row_data = w.data + tile.group * w.matrix_bytes + my_row * w.row_bytes;
    row_scales = tile.group * w.scales_matrix_stride + my_row * w.scale_stride;
  } else {
    row_data = static_cast<const uint8_t*>(c.lhs) + (tile.group * c.matrix_stride + my_row * c.lhs_rs) * T::kBytes;
  }
  const int row_bytes = kInt4 ? (c.k + 1) / 2 : c.k * T::kBytes;
  const int row_scale_count = kInt4 ? (c.k + w.group_size - 1) / w.group_size : 0;
  const bool f32_scales = w.scale_type == RUYAMD_DTYPE_F32;

  struct Held {
    v4i weights[T::kWeightLoads];
    uint32_t scales[kScales], zeros[kScales];  // (Scaling::kAny)
  };
  // Loads never reach past the end of a row (which has 16 bytes at least): what would is
  // read from its last bytes, and moved to where it belongs by Place.
  const auto load = [&](int chunk, Held& h) __attribute__((always_inline)) {
    if constexpr (kInt4 && !kScalesInLds) {
#pragma unroll
      for (int g = 0; g < kScales; ++g) {
        const int at = min(chunk * T::kChunk + g * (T::kChunk / kScales), c.k - 1) / w.group_size;
        h.scales[g] = f32_scales ? static_cast<const uint32_t*>(w.scales)[row_scales + at]
                                 : static_cast<const uint16_t*>(w.scales)[row_scales + at];
        h.zeros[g] = kZeroPoints ? w.zero_points[row_scales + at] : 8;
      }
    }
#pragma unroll
    for (int i = 0; i < T::kWeightLoads; ++i) {
      const int at = min(chunk * (T::kWeightLoads * 64) + i * 64 + q * 16, row_bytes - 16);
      h.weights[i] = *reinterpret_cast<const granule::v4i_unaligned*>(row_data + at);
    }
  };
  const auto place = [&](int chunk, Held& h) __attribute__((always_inline)) {
    if (chunk < whole_chunks) return;
#pragma unroll
    for (int i = 0; i < T::kWeightLoads; ++i) {
      const int at = chunk * (T::kWeightLoads * 64) + i * 64 + q * 16;
      h.weights[i] = granule::PlaceGranule(h.weights[i], at, row_bytes);
    }
  };
  // A scale's bits, read as its type, as a number.
  const auto as_float = [&](uint32_t bits) __attribute__((always_inline)) -> float {
    const float as_half = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
    const float as_bf16 = __uint_as_float(bits << 16), as_is = __uint_as_float(bits);
    return f32_scales ? as_is : w.scale_type == RUYAMD_DTYPE_BF16 ? as_bf16 : as_half;
  };
  // Scales and zero points of a workgroup's rows are put into LDS first, as numbers and zeros behind
  // the last. (Where they lie they are 2 bytes of a line that has gone from the caches when the
  // next 2 are wanted: 16384 x 16384 half, one token, 36 us with scales read
  // where they lie, 29.7 with these.)
  const float* const lds_scales = reinterpret_cast<const float*>(lds + args.scales_at);
  const uint8_t* const lds_zeros = reinterpret_cast<const uint8_t*>(lds + args.zeros_at);
  const auto put_scales = [&]() __attribute__((always_inline)) {
    if constexpr (kScalesInLds) {
      const int padded = chunks * kScales, all_waves = depth_waves * row_waves;
      float* const to = reinterpret_cast<float*>(lds + args.scales_at);
      uint8_t* const zeros_to = reinterpret_cast<uint8_t*>(lds + args.zeros_at);
      constexpr int kAtOnce = 4;
      for (int row = wave * kAtOnce; row < work_rows; row += all_waves * kAtOnce)
        for (int g = lane; g < padded; g += 64) {
          uint32_t bits[kAtOnce], zeros[kAtOnce];
          // (A scale that several chunks share is there several times.)
          const int at = kScaling == Scaling::kWide ? static_cast<int>(int64_t(g) * 128 >> args.scale_shift) : g;
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) {
            const int64_t from = tile.group * w.scales_matrix_stride + min(row0 + row + i, c.m - 1) * w.scale_stride + at;
            bits[i] = zeros[i] = 0;
            if (at < row_scale_count) {
              bits[i] = f32_scales ? static_cast<const uint32_t*>(w.scales)[from] : static_cast<const uint16_t*>(w.scales)[from];
              if constexpr (kZeroPoints) zeros[i] = w.zero_points[from];
            }
          }
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) {
            to[(row + i) * args.scale_pitch + g] = as_float(bits[i]);
            if constexpr (kZeroPoints) zeros_to[(row + i) * args.zero_pitch + g] = static_cast<uint8_t>(zeros[i]);
          }
        }
    }
  };
  const auto scales_of = [&](const Held& h, int chunk, float (&scale)[kScales], uint32_t (&zero)[kScales])
                             __attribute__((always_inline)) {
    const int row = row_wave * 16 + l;
#pragma unroll
    for (int g = 0; g < kScales; ++g) {
      scale[g] = kScalesInLds ? lds_scales[row * args.scale_pitch + chunk * kScales + g] : as_float(h.scales[g]);
      zero[g] = 8;
      if constexpr (kZeroPoints)
        zero[g] = kScalesInLds ? lds_zeros[row * args.zero_pitch + chunk * kScales + g] : h.zeros[g];
    }
  };

  // Unit u of a token (kUnit values from depth position u * kUnit on), zeros past the depth.
  struct Unit {
    v4i x[T::kUnitLoads];
  };
  const uint8_t* const token_data =
      static_cast<const uint8_t*>(c.rhs) + (int64_t(range.begin) + token0) * c.rhs_cs * T::kBytes;
  // (One inside the depth, of tokens whose values lie side by side.)
  const auto fetch_inside = [&](int token, int u) __attribute__((always_inline)) -> Unit {
    Unit unit;
    const uint8_t* p = token_data + (token * c.rhs_cs + u * T::kUnit) * T::kBytes;
#pragma unroll
    for (int i = 0; i < T::kUnitLoads; ++i) unit.x[i] = reinterpret_cast<const granule::v4i_unaligned*>(p)[i];
    return unit;
  };
  const auto fetch = [&](int token, int u) __attribute__((always_inline)) -> Unit {
    Unit unit;
    const int k = u * T::kUnit;
    constexpr int kValues = 16 / T::kBytes;
    if (c.rhs_rs == 1) {
      const uint8_t* p = token_data + token * c.rhs_cs * T::kBytes;
#pragma unroll
      for (int i = 0; i < T::kUnitLoads; ++i) {
        const int at = (k + i * kValues) * T::kBytes;
        unit.x[i] = granule::PlaceGranule(granule::LoadGranule<false>(p, at, c.k * T::kBytes), at, c.k * T::kBytes);
      }
      return unit;
    }
    const uint8_t* p = token_data + (token * c.rhs_cs + k * c.rhs_rs) * T::kBytes;
#pragma unroll
    for (int i = 0; i < T::kUnitLoads; ++i) {
      v4i x = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < kValues; ++e) {
        const int at = i * kValues + e;
        if (k + at >= c.k) continue;
        if constexpr (T::kBytes == 4)
          x[e] = *reinterpret_cast<const int*>(p + at * c.rhs_rs * 4);
        else
          x[e / 2] |= static_cast<int>(uint32_t(*reinterpret_cast<const uint16_t*>(p + at * c.rhs_rs * 2)) << (16 * (e & 1)));
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
  // The remainders that the third parts of this lane's tokens were rounded from (float_parts::Lost), and whether a wave
  // has had a token that is not its parts' sum: one for all waves, whichever has taken it apart.
  int lost = 0;
  int* const lds_lost = reinterpret_cast<int*>(lds + args.lost_at);
  const auto put_lost = [&]() __attribute__((always_inline)) {
    if constexpr (T::kParts) {
      const bool any = __any(float_parts::Lost(lost)) != 0;
      if (lane == 0) lds_lost[wave] = any;
    }
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
        lost |= __float_as_int(x) | __float_as_int(y);
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

  v4f acc[kCols] = {};

  // What the eight values of a word are taken apart with. (Held in registers: as constants
  // in the instructions they would each take one more.)
  uint32_t low_mask = 0x000F000Fu, high_mask = 0x00F000F0u, sixteenth = 0x2C002C00u, exponent = 0x64006400u;
  asm("" : "+s"(low_mask));
  asm("" : "+s"(high_mask));
  asm("" : "+s"(sixteenth));
  asm("" : "+v"(exponent));
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  const auto halves = [](uint32_t x) __attribute__((always_inline)) -> v2h { return __builtin_bit_cast(v2h, x); };
  const auto bits = [](v2h x) __attribute__((always_inline)) -> int { return __builtin_bit_cast(int, x); };
  // Half: q - zero, in the order 0 4 1 5 2 6 3 7. 1024 + q (its four bits lowest in the mantissa) less 1024 + zero, or
  // 1024 + 16 q (one place further up) sixteenths less 64 + zero; all exact.
  const auto less_zero = [&](uint32_t x, uint32_t zero) __attribute__((always_inline)) -> v4i {
    const uint32_t low = 0x6400u | zero, high = 0xD400u | zero << 4;  // 1024 + zero, -(64 + zero)
    const v2h away_low = halves(low | low << 16), away_high = halves(high | high << 16);
    const uint32_t y = x >> 8;
    return v4i{bits(halves((x & low_mask) | exponent) - away_low),
               bits(__builtin_elementwise_fma(halves((x & high_mask) | exponent), halves(sixteenth), away_high)),
               bits(halves((y & low_mask) | exponent) - away_low),
               bits(__builtin_elementwise_fma(halves((y & high_mask) | exponent), halves(sixteenth), away_high))};
  };
  // The same as bfloat16, exact too (whole numbers of 4 bits and a sign). The factors are variables: a product with a half
  // and a sum are one instruction then, a conversion and a sum two.
  float whole_factor = 1.0f, sixteenth_factor = 0.0625f;
  asm("" : "+v"(whole_factor));
  asm("" : "+v"(sixteenth_factor));
  const auto less_zero_bf16 = [&](uint32_t x, uint32_t zero) __attribute__((always_inline)) -> v4i {
    const float z = static_cast<float>(zero), away_low = -1024.0f - z, away_high = -64.0f - z;
    const auto less = [&](uint32_t with_exponent, float factor, float away) __attribute__((always_inline)) -> int {
      const v2h pair = halves(with_exponent);
      const float first = __builtin_fmaf(static_cast<float>(pair[0]), factor, away);
      const float second = __builtin_fmaf(static_cast<float>(pair[1]), factor, away);
      return static_cast<int>(__builtin_amdgcn_perm(__float_as_uint(second), __float_as_uint(first), 0x07060302));
    };
    const uint32_t y = x >> 8;
    return v4i{less((x & low_mask) | exponent, whole_factor, away_low),
               less((x & high_mask) | exponent, sixteenth_factor, away_high),
               less((y & low_mask) | exponent, whole_factor, away_low),
               less((y & high_mask) | exponent, sixteenth_factor, away_high)};
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
    return kInt4 && kScaling == Scaling::kWide ? j / 4 * 16 + q * 4 + j % 4 : j * 4 + q;
  };

  // `at`: the chunk's place in the tokens' rows.
  const auto use = [&](const Held& h, int chunk, const char* at) __attribute__((always_inline)) {
    if constexpr (!kInt4) {
#pragma unroll
      for (int j = 0; j < T::kSteps; ++j)
#pragma unroll
        for (int t = 0; t < kCols; ++t) {
          const v4i x = *reinterpret_cast<const v4i*>(at + lds_row[t] * args.pitch + unit_of(j) * 16);
          Mma<kType>(x, h.weights[j], acc[t]);
        }
    } else {
      v4i words[T::kWeightLoads];
      float scale[kScales];
      uint32_t zero[kScales];
      scales_of(h, chunk, scale, zero);
#pragma unroll
      for (int i = 0; i < T::kWeightLoads; ++i) words[i] = exchange(h.weights[i]);
#pragma unroll
      for (int g = 0; g < kScales; ++g) {
        v4f sum[kCols] = {};
#pragma unroll
        for (int f = 0; f < kStepsToScale; ++f) {
          const int j = g * kStepsToScale + f;
          v4i x[kCols];
#pragma unroll
          for (int t = 0; t < kCols; ++t)
            x[t] = *reinterpret_cast<const v4i*>(at + lds_row[t] * args.pitch + unit_of(j) * 16);
          const uint32_t word = words[j / 4][j % 4];
          const v4i b = kHalf ? less_zero(word, zero[g]) : less_zero_bf16(word, zero[g]);
#pragma unroll
          for (int t = 0; t < kCols; ++t) Mma<kMmaType>(x[t], b, sum[t]);
        }
#pragma unroll
        for (int t = 0; t < kCols; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][e] = __builtin_fmaf(scale[g], sum[t][e], acc[t][e]);
      }
    }
  };

  constexpr int kLdsChunk = T::kChunkUnits * 16;
  // Turns of this wave's main loop, a whole chunk each; the slabs' turns are those of all
  // waves. What is left of the depth comes behind the loop.
  const int turns = kSlabs ? whole_chunks / depth_waves
                           : (whole_chunks - depth_wave + depth_waves - 1) / depth_waves;
  // The depth begins at another place in every 16 rows and goes round: rows
  // often lie a power of two apart, and whoever goes through theirs side by side, from
  // the same place on, asks the same few memory channels. (Places by a multiplicative hash; one after
  // the other they meet again at some row lengths. 16384 rows of 8 KiB read alone, 4 waves
  // along the depth: the same place 28 us, one after the other 33, hashed 25.7.)
  const uint32_t unit = (static_cast<uint32_t>(tile.group) * args.tiles_m + tile.m) * row_waves + (kSlabs ? 0 : row_wave);
  const int first_turn = turns > 0 ? static_cast<int>((unit * 2654435761u >> 12) % static_cast<uint32_t>(turns)) : 0;
  const auto place_of = [&](int turn) __attribute__((always_inline)) -> int {  // (past the last: the last)
    const int at = min(turn, turns - 1) + first_turn;
    return at < turns ? at : at - turns;
  };
  // The loop's loads are issued whatever comes (past the end once more the last chunk):
  // a load that may or may not have been issued is one for which everything is waited for.
  Held held[2], last;
  const bool has_last = !kSlabs && whole_chunks < chunks && (whole_chunks & (depth_waves - 1)) == depth_wave;
  if (has_last) load(whole_chunks, last);
  if (turns > 0) {
    load(depth_wave + place_of(0) * depth_waves, held[0]);
    load(depth_wave + place_of(1) * depth_waves, held[1]);
  }
  put_scales();
  if constexpr (kSlabs) {
    const int slab_units = depth_waves * T::kChunkUnits, unit_bits = __builtin_ctz(slab_units);  // (a power of two)
    constexpr int kPieces = (kMostTokens * T::kChunkUnits + 64 * kRowWaves - 1) / (64 * kRowWaves);
    Unit pieces[kPieces];  // the next slab, on its way
    // (Tokens past the last are the last one again.)
    const auto fetch_slab = [&](int slab) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int n = i * blockDim.x + threadIdx.x, token = min(n >> unit_bits, tokens - 1);
        pieces[i] = fetch_inside(token, slab * slab_units + (n & (slab_units - 1)));
      }
    };
    const auto put_slab = [&](int buffer) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int n = i * blockDim.x + threadIdx.x, token = min(n >> unit_bits, tokens - 1);
        put(pieces[i], lds + buffer * args.slab_bytes + row_in_lds(token) * args.pitch + (n & (slab_units - 1)) * 16);
      }
    };
    if (turns > 0) {
      fetch_slab(place_of(0));
      put_slab(0);
      fetch_slab(place_of(1));
      const auto turn = [&](int n, auto d) __attribute__((always_inline)) {
        // Slab n is there, and slab n - 1 no longer read, when all have come here.
        __syncthreads();
        put_slab(1 - d);
        fetch_slab(place_of(n + 2));
        use(held[d], depth_wave + place_of(n) * depth_waves, lds + d * args.slab_bytes + depth_wave * kLdsChunk);
        load(depth_wave + place_of(n + 2) * depth_waves, held[d]);
      };
      for (int n = 0;;) {
        turn(n, std::integral_constant<int, 0>());
        if (++n == turns) break;
        turn(n, std::integral_constant<int, 1>());
        if (++n == turns) break;
      }
    }
    const int done = turns * depth_waves, left = chunks - done;
    if (left > 0) {
      __syncthreads();
      const int units = left * T::kChunkUnits;
      for (int n = threadIdx.x; n < tokens * units; n += blockDim.x)
        put(fetch(n / units, done * T::kChunkUnits + n % units), lds + row_in_lds(n / units) * args.pitch + n % units * 16);
      __syncthreads();
      if (depth_wave < left) {
        load(done + depth_wave, held[0]);
        place(done + depth_wave, held[0]);
        use(held[0], done + depth_wave, lds + depth_wave * kLdsChunk);
      }
    }
    if constexpr (T::kParts) {
      put_lost();
      __syncthreads();
    }
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
    put_lost();
    __syncthreads();
    if (turns > 0) {
      const auto turn = [&](int n, auto d) __attribute__((always_inline)) {
        const int chunk = depth_wave + place_of(n) * depth_waves;
        use(held[d], chunk, lds + chunk * kLdsChunk);
        load(depth_wave + place_of(n + 2) * depth_waves, held[d]);
      };
      for (int n = 0;;) {
        turn(n, std::integral_constant<int, 0>());
        if (++n == turns) break;
        turn(n, std::integral_constant<int, 1>());
        if (++n == turns) break;
      }
    }
    if (has_last) {
      place(whole_chunks, last);
      use(last, whole_chunks, lds + whole_chunks * kLdsChunk);
    }
  }

  if constexpr (T::kParts) {
    bool again = false;
#pragma unroll
    for (int t = 0; t < kCols; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) again = again || !__builtin_isfinite(acc[t][e]);
    if (lane < depth_waves * row_waves) again = again || lds_lost[lane] != 0;
    if (__any(again)) {
      // Once more, with whole tokens on the fp32 instructions.
#pragma unroll
      for (int t = 0; t < kCols; ++t) acc[t] = v4f{0, 0, 0, 0};
#pragma unroll 1
      for (int chunk = depth_wave; chunk < chunks; chunk += depth_waves) {
        Held h;
        load(chunk, h);
        place(chunk, h);
        float scale[kScales];
        uint32_t zero[kScales];
        scales_of(h, chunk, scale, zero);
#pragma unroll
        for (int i = 0; i < T::kWeightLoads; ++i) h.weights[i] = exchange(h.weights[i]);
#pragma unroll
        for (int g = 0; g < kScales; ++g) {
#pragma unroll 1
          for (int f = 0; f < kStepsToScale; ++f) {
            const int j = g * kStepsToScale + f;
#pragma unroll
            for (int t = 0; t < kCols; ++t) {
              // (The whole token in the place of its first part.)
              const int token = min(t * T::kTokens + l / 3, tokens - 1);
              const Unit x = fetch(token, chunk * T::kChunkUnits + unit_of(j));
              const uint32_t word = h.weights[g * kStepsToScale / 4][0];
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(static_cast<int>(word >> (4 * e) & 15) - static_cast<int>(zero[g]));
              v4f sum = {0, 0, 0, 0};
#pragma unroll
              for (int e = 0; e < 8; ++e)
                sum = __builtin_amdgcn_mfma_f32_16x16x4f32(l % 3 == 0 ? __int_as_float(x.x[e / 4][e % 4]) : 0.0f, v[e], sum,
                                                           0, 0, 0);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[t][e] = __builtin_fmaf(scale[g], sum[e], acc[t][e]);
            }
            // (The next step's word in the place of this one's.)
            v4i& x = h.weights[g * kStepsToScale / 4];
            x = v4i{x[1], x[2], x[3], 0};
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
    for (int e = 0; e < 4; ++e) partial[(wave * 4 + e) * 64 + lane] = acc[t][e];
    __syncthreads();
    // Value number v: row v % 16 of a block of 16, token v / 16 % 16, block v / 256.
    for (int v = threadIdx.x; v < work_rows * T::kTokens; v += blockDim.x) {
      const int row = v % 16, token = v / 16 % T::kTokens, r = v / (16 * T::kTokens);
      const int m = row0 + r * 16 + row, n = token0 + t * T::kTokens + token;
      if (m >= c.m || n >= token0 + tokens) continue;
      float sum = 0;
#pragma unroll
      for (int s = 0; s < (T::kParts ? 3 : 1); ++s) {
        const int at = T::kParts ? token * 3 + s : token;  // row of the accumulators' block
        const float* from = partial + (r * 4 + at % 4) * 64 + at / 4 * 16 + row;
        for (int i = 0; i < depth_waves; ++i) sum += from[i * row_waves * 256];
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
  int cols;  // kCols of the kernel
  bool slabs;
  Scaling scaling;
  unsigned lds_bytes;
};

template <bool kInt4, int kType, int kCols, Scaling kScaling, bool kSlabs, bool kZeroPoints>
hipError_t LaunchStreamKernel(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  auto* const kernel = &GroupedStreamKernel<kInt4, kType, kCols, kScaling, kSlabs, kZeroPoints>;
  static const hipError_t attribute = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, kStreamLds);
  if (attribute != hipSuccess) return attribute;
  hipLaunchKernelGGL(kernel, dim3(plan.blocks), dim3(64 * plan.waves), plan.lds_bytes, stream, args);
  return hipGetLastError();
}

template <int kType, Scaling kScaling, bool kZeroPoints>
hipError_t LaunchStreamInt4Of(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  if (plan.cols == 2)
    return LaunchStreamKernel<true, kType, 2, kScaling, true, kZeroPoints>(stream, args, plan);
  if (plan.slabs)
    return LaunchStreamKernel<true, kType, 1, kScaling, true, kZeroPoints>(stream, args, plan);
  return LaunchStreamKernel<true, kType, 1, kScaling, false, kZeroPoints>(stream, args, plan);
}

template <int kType, Scaling kScaling>
hipError_t LaunchStreamScaling(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  if (args.w.zero_points) return LaunchStreamInt4Of<kType, kScaling, true>(stream, args, plan);
  return LaunchStreamInt4Of<kType, kScaling, false>(stream, args, plan);
}

template <int kType>
hipError_t LaunchStreamInt4(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  switch (plan.scaling) {
    case Scaling::kWide:
      return LaunchStreamScaling<kType, Scaling::kWide>(stream, args, plan);
    case Scaling::k64:
      return LaunchStreamScaling<kType, Scaling::k64>(stream, args, plan);
    case Scaling::k32:
      return LaunchStreamScaling<kType, Scaling::k32>(stream, args, plan);
    default:
      return LaunchStreamScaling<kType, Scaling::kAny>(stream, args, plan);
  }
}

// Weights in the tokens' type.
template <int kType>
hipError_t LaunchStreamFloat(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  if (plan.cols == 2)
    return LaunchStreamKernel<false, kType, 2, Scaling::kWide, true, false>(stream, args, plan);
  if (plan.slabs)
    return LaunchStreamKernel<false, kType, 1, Scaling::kWide, true, false>(stream, args, plan);
  return LaunchStreamKernel<false, kType, 1, Scaling::kWide, false, false>(stream, args, plan);
}

// (Each in a file of its own.)
hipError_t LaunchStreamInt4Bf16(hipStream_t, const StreamArgs&, const StreamPlan&);
hipError_t LaunchStreamInt4F16(hipStream_t, const StreamArgs&, const StreamPlan&);
hipError_t LaunchStreamInt4F32(hipStream_t, const StreamArgs&, const StreamPlan&);

}  // namespace grouped
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_GROUPED_STREAM_H_
