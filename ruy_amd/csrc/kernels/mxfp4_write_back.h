// The write-back of the tiled kernels for 4-bit values.
#ifndef RUY_AMD_CSRC_KERNELS_MXFP4_WRITE_BACK_H_
#define RUY_AMD_CSRC_KERNELS_MXFP4_WRITE_BACK_H_

#include "grouped_device.h"
#include "mxfp4_device.h"

namespace ruyamd {
namespace mxfp4 {

// A wave has kBlocksM x kBlocksN blocks of 16x16: lane l holds column l % 16 of a block and, of the blocks number 2 i and
// 2 i + 1 along the rows, rows (l / 16) * 8 .. + 7 of 32. They go to dst's rows from m0 on (`rows` of them are there, maybe none
// or less) and columns from n0 on; `bias` is of the first row.
//
// A lone wave on its SIMD waits for whatever it waits for, and goes through most of this once: what matters is few instructions,
// in loops where they are long, and none that waits for the one before. Types and edges told apart for every block in
// place made 200 KB of instructions: 22 us for a 256x256 tile in 16 bits. Stores past
// the caches gained nothing.
template <int kBlocksM, int kBlocksN>
struct WriteBack {
  static constexpr int kRows = kBlocksM * 16, kColumns = kBlocksN * 16;
  static constexpr int kLanes = kRows / 8, kAtOnce = 64 / kLanes;  // lanes to a column of 8 rows each, columns at once
  static constexpr int kPitch16 = kRows * 2 + 16;                  // bytes from a column to the next in LDS, 16-bit values
  static constexpr int kPitch32 = kRows * 4 + 16, kColumns32 = 32; // and fp32 ones, fewer at a time
  static constexpr int kLds = kColumns * kPitch16 > kColumns32 * kPitch32 ? kColumns * kPitch16 : kColumns32 * kPitch32;  // a wave's
  typedef __attribute__((aligned(2))) v4i v4i_of_2;
  typedef __attribute__((aligned(4))) v4f v4f_of_4;
  using Blocks = v4f[kBlocksM][kBlocksN];

  const MulCall& c;
  const Blocks& acc;
  char* const lds;
  const float* const bias;
  const int64_t m0, n0;
  const int rows, columns;
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;

  // The 8 values of blocks 2 i, 2 i + 1 and column block j.
  template <bool kPlain>
  __device__ __forceinline__ void Values(int i, int j, const float (&add)[8], float (&v)[8]) const {
    // (Held to this place: what the variants have in common the compiler would otherwise do for all blocks at once in front of them, in
    // more registers than there are.)
    v4f low = acc[2 * i][j], high = acc[2 * i + 1][j];
    asm volatile("" : "+v"(low), "+v"(high));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = e < 4 ? low[e & 3] : high[e & 3];
      // (Of a NaN these leave a NaN, as grouped::Clamp.)
      if constexpr (!kPlain) v[e] = __builtin_elementwise_maximum(__builtin_elementwise_minimum(v[e] + add[e], c.clamp_max), c.clamp_min);
    }
  }
  // The bias of a lane's rows, all of it on its way at once.
  struct Added {
    float of[kBlocksM / 2][8];
  };
  template <bool kPlain>
  __device__ __forceinline__ Added Bias() const {
    Added add = {};
    if (!kPlain && bias) {
#pragma unroll
      for (int i = 0; i < kBlocksM / 2; ++i) {
        const int m = i * 32 + q * 8;
        if (m + 8 <= rows) {
          const v4f low = *reinterpret_cast<const v4f_of_4*>(bias + m), high = *reinterpret_cast<const v4f_of_4*>(bias + m + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e) add.of[i][e] = e < 4 ? low[e & 3] : high[e & 3];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (m + e < rows) add.of[i][e] = bias[m + e];
        }
      }
    }
    return add;
  }

  // 16-bit values by columns: rounded where they are, and through LDS, so that whole lines of dst are stored.
  template <bool kPlain>
  __device__ __forceinline__ void Half() const {
    const bool bf16 = c.dst_type == RUYAMD_DTYPE_BF16;
    const Added add = Bias<kPlain>();
#pragma unroll
    for (int i = 0; i < kBlocksM / 2; ++i) {
      float v[8];
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) {
        Values<kPlain>(i, j, add.of[i], v);
        v4i packed;
        if (bf16) {
#pragma unroll
          for (int e = 0; e < 4; ++e) packed[e] = grouped::RoundPair<RUYAMD_DTYPE_BF16>(v[2 * e], v[2 * e + 1]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) packed[e] = grouped::RoundPair<RUYAMD_DTYPE_F16>(v[2 * e], v[2 * e + 1]);
        }
        *reinterpret_cast<v4i*>(lds + (j * 16 + l) * kPitch16 + i * 64 + q * 16) = packed;
      }
    }
    __builtin_amdgcn_wave_barrier();  // (A wave's own part of LDS: its accesses stay in order.)
    const int m = lane % kLanes * 8;
    const char* const from = lds + lane / kLanes * kPitch16 + m * 2;
    uint16_t* const to = static_cast<uint16_t*>(c.dst) + (n0 + lane / kLanes) * c.dst_cs + m0 + m;
    constexpr int kUnroll = kColumns / kAtOnce < 8 ? kColumns / kAtOnce : 8;
#pragma unroll 1
    for (int n = 0; n < kColumns; n += kUnroll * kAtOnce) {
      v4i held[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) held[u] = *reinterpret_cast<const v4i*>(from + (n + u * kAtOnce) * kPitch16);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int column = n + u * kAtOnce;
        if (column + lane / kLanes >= columns) continue;
        if (m + 8 <= rows) {
          *reinterpret_cast<v4i_of_2*>(to + column * c.dst_cs) = held[u];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (m + e < rows) to[column * c.dst_cs + e] = static_cast<uint16_t>(static_cast<uint32_t>(held[u][e / 2]) >> (16 * (e & 1)));
        }
      }
    }
  }

  // fp32 by columns, all rows: four lanes' 32 bytes are a whole line.
  template <bool kPlain>
  __device__ __forceinline__ void Full() const {
    const Added add = Bias<kPlain>();
#pragma unroll
    for (int i = 0; i < kBlocksM / 2; ++i) {
      float v[8];
#pragma unroll
      for (int j = 0; j < kBlocksN; ++j) {
        Values<kPlain>(i, j, add.of[i], v);
        if (j * 16 + l >= columns) continue;
        v4f_of_4* const p = reinterpret_cast<v4f_of_4*>(static_cast<float*>(c.dst) + (n0 + j * 16 + l) * c.dst_cs + m0 + i * 32 + q * 8);
        p[0] = v4f{v[0], v[1], v[2], v[3]};
        p[1] = v4f{v[4], v[5], v[6], v[7]};
      }
    }
  }

  // Anything else: value by value, out of LDS in a loop; lanes along the columns, which is how dst by rows lies. (us, bfloat16 by columns and
  // by rows: 8192 x 8192 x 512 48 and 129, 4096 x 4096 x 4096 38 and 76, 8192 x 8192 x 8192 275 and 398; fp32 by columns, 4096 rows 43 and
  // 4000, whose last tile is cut short, 59.)
  __device__ __forceinline__ void Each() const {
    constexpr int kBlocks = kColumns32 / 16;
    const float* const held = reinterpret_cast<const float*>(lds);
#pragma unroll
    for (int j0 = 0; j0 < kBlocksN; j0 += kBlocks) {
#pragma unroll
      for (int j = 0; j < kBlocks; ++j)
#pragma unroll
        for (int i = 0; i < kBlocksM; ++i) {
          v4f x = acc[i][j0 + j];
          asm volatile("" : "+v"(x));
          *reinterpret_cast<v4f*>(lds + (j * 16 + l) * kPitch32 + ((i >> 1) * 32 + q * 8 + (i & 1) * 4) * 4) = x;
        }
      __builtin_amdgcn_wave_barrier();
      const int n = lane % kColumns32;
#pragma unroll 4
      for (int m = lane / kColumns32; m < kRows; m += 64 / kColumns32) {
        const float v = held[n * (kPitch32 / 4) + m];
        if (m < rows && j0 * 16 + n < columns)
          grouped::StoreFloat(c.dst, c.dst_type, (n0 + j0 * 16 + n) * c.dst_cs + (m0 + m) * c.dst_rs,
                              grouped::Clamp(v + (bias ? bias[m] : 0.0f), c.clamp_min, c.clamp_max));
      }
      __builtin_amdgcn_wave_barrier();
    }
  }

  template <bool kPlain>
  __device__ __forceinline__ void Columns() const {
    if (c.dst_type == RUYAMD_DTYPE_F32)
      Full<kPlain>();
    else
      Half<kPlain>();
  }
  __device__ __forceinline__ void operator()() const {
    if (c.dst_rs != 1 || (c.dst_type == RUYAMD_DTYPE_F32 && rows < kRows)) return Each();
    const float infinity = __uint_as_float(0x7f800000u);
    if (!bias && c.clamp_max == infinity && c.clamp_min == -infinity) return Columns<true>();
    Columns<false>();
  }
};

}  // namespace mxfp4
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_MXFP4_WRITE_BACK_H_
