// Values to 4 bits with a power of two to each block, and back
// (ruyamd_quantize_mxfp4, ruyamd_dequantize_mxfp4).
//
// A lane has 8 values of a row, and four neighbours a block: its largest magnitude is found by two
// exchanges between them. Both directions are a copy of what they read and write: 8 values come or go
// as 16 or 32 bytes, their 4-bit numbers as one word, a block's scale as a byte.
//
// v_cvt_scalef32_pk_fp4_f32 rounds to nearest, ties to even, and holds what is larger to 6, as OCP MX 1.0 says; it is given the values
// already divided by their power of two, which is exact but for what is far too small to become anything but 0. HBM bounds both
// directions: 8192 x 4096 bfloat16 values 67 + 18 MB, into two places each 22.5 us (4.6 TB/s) and one matrix of twice the rows back 26.6
// (6.5); a ragged one of 1000 x 1500 fp32 values 3.7 and 4.4 us, which are launch and latency.
#include <algorithm>

#include "granule.h"
#include "grouped_device.h"
#include "launch_geometry.h"
#include "mxfp4_device.h"

namespace ruyamd {
namespace mxfp4 {
namespace {

using granule::v4i;
using granule::v4i_unaligned;
using grouped::LoadFloat;
using grouped::RoundPair;
using grouped::StoreFloat;

typedef uint32_t u32_unaligned __attribute__((aligned(1)));

constexpr int Bytes(int type) { return type == RUYAMD_DTYPE_F32 ? 4 : 2; }

// A row and which of its segments of 64 * kUnits units of 8 values this wave has.
struct Piece {
  int row, segment;
};
__device__ __forceinline__ int64_t FirstPiece() {
  return int64_t(blockIdx.x) * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}
__device__ __forceinline__ int64_t PieceStride() { return int64_t(gridDim.x) * (blockDim.x >> 6); }
__device__ __forceinline__ Piece PieceOf(int64_t i, int segments) {
  const int row = static_cast<int>(i / segments);
  return {row, static_cast<int>(i - int64_t(row) * segments)};
}

// f(row of the matrix) for every place that a row goes to.
template <class F>
__device__ __forceinline__ void ForEachPlace(const ConvertCall& c, int row, F&& f) {
  if (!c.places) return f(row);
  for (int j = 0; j < c.top; ++j) {
    const int p = c.places[int64_t(row) * c.top + j];
    if (p >= 0 && p < c.matrix.rows) f(p);
  }
}

// 8 values as they lie, and as numbers.
template <int kType>
struct Unit {
  static constexpr int kGranules = 8 * Bytes(kType) / 16;
  v4i raw[kGranules];

  __device__ __forceinline__ void Load(const char* row, int64_t first) {
#pragma unroll
    for (int i = 0; i < kGranules; ++i) raw[i] = reinterpret_cast<const v4i_unaligned*>(row + first * Bytes(kType))[i];
  }
  __device__ __forceinline__ void Values(float (&v)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (kType == RUYAMD_DTYPE_F32) {
        v[e] = __int_as_float(raw[e / 4][e % 4]);
      } else {
        const uint32_t word = static_cast<uint32_t>(raw[0][e / 2]);
        if constexpr (kType == RUYAMD_DTYPE_BF16)
          v[e] = __uint_as_float(e % 2 ? word & 0xffff0000u : word << 16);
        else
          v[e] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(e % 2 ? word >> 16 : word)));
      }
    }
  }
  __device__ __forceinline__ void Store(char* row, int64_t first, const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < kGranules; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kType == RUYAMD_DTYPE_F32)
          raw[i][e] = __float_as_int(v[i * 4 + e]);
        else
          raw[i][e] = RoundPair<kType>(v[2 * e], v[2 * e + 1]);
      }
      reinterpret_cast<v4i_unaligned*>(row + first * Bytes(kType))[i] = raw[i];
    }
  }
};

// The largest over each four neighbouring lanes.
__device__ __forceinline__ uint32_t LargestOfFour(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xb1, 0xf, 0xf, true)));  // lanes 1 0 3 2
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4e, 0xf, 0xf, true)));  // lanes 2 3 0 1
  return v;
}

template <int kType, int kUnits>
__global__ __launch_bounds__(256) void QuantizeKernel(ConvertCall c, int segments) {
  const int lane = threadIdx.x & 63, cols = c.matrix.cols;
  const int64_t pieces = int64_t(c.rows) * segments;
  for (int64_t i = FirstPiece(); i < pieces; i += PieceStride()) {
    const Piece piece = PieceOf(i, segments);
    const char* const from = static_cast<const char*>(c.data) + piece.row * c.rs * Bytes(kType);
    const int64_t unit0 = int64_t(piece.segment) * (64 * kUnits) + lane;
    // (All of the segment inside the row, the same for all lanes: its loads go out together.)
    const bool whole = (int64_t(piece.segment) + 1) * (512 * kUnits) <= cols;
    float v[kUnits][8];
    uint32_t packed[kUnits];
    int scale[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = 0;
    }
    if (whole) {
      Unit<kType> held[kUnits];
#pragma unroll
      for (int u = 0; u < kUnits; ++u) held[u].Load(from, (unit0 + u * 64) * 8);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) held[u].Values(v[u]);
    } else {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int64_t first = (unit0 + u * 64) * 8;
        if (first + 8 <= cols) {
          Unit<kType> held;
          held.Load(from, first);
          held.Values(v[u]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (first + e < cols) v[u][e] = LoadFloat(from, kType, first + e);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      uint32_t largest = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) largest = max(largest, __float_as_uint(v[u][e]) & 0x7fffffffu);
      scale[u] = ScaleOf(LargestOfFour(largest));
      const float inverse = InverseOf(scale[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] *= inverse;
      packed[u] = scale[u] == kNaNScale ? 0 : Round8(v[u]);
    }
    // Lane 4 b + u stores the scale of unit u's block b.
    int my_scale = scale[0];
#pragma unroll
    for (int u = 1; u < kUnits; ++u) my_scale = (lane & 3) == u ? scale[u] : my_scale;
    const int64_t my_block = int64_t(piece.segment) * (16 * kUnits) + (lane & 3) * 16 + (lane >> 2);
    ForEachPlace(c, piece.row, [&](int row) __attribute__((always_inline)) {
      uint8_t* const data = c.matrix.data + row * c.matrix.row_bytes;
      uint8_t* const scales = c.matrix.scales + row * c.matrix.scale_stride;
      if ((lane & 3) < kUnits && my_block * kBlock < cols) scales[my_block] = static_cast<uint8_t>(my_scale);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int64_t first = (unit0 + u * 64) * 8;
        if (whole || first + 8 <= cols) {
          *reinterpret_cast<u32_unaligned*>(data + first / 2) = packed[u];
        } else if (first < cols) {
          for (int b = 0; b < (cols - first + 1) / 2; ++b) data[first / 2 + b] = static_cast<uint8_t>(packed[u] >> (8 * b));
        }
      }
    });
  }
}

template <int kType, int kUnits>
__global__ __launch_bounds__(256) void DequantizeKernel(ConvertCall c, int segments) {
  const int lane = threadIdx.x & 63, cols = c.matrix.cols;
  const int64_t pieces = int64_t(c.rows) * segments;
  for (int64_t i = FirstPiece(); i < pieces; i += PieceStride()) {
    const Piece piece = PieceOf(i, segments);
    const uint8_t* const data = c.matrix.data + piece.row * c.matrix.row_bytes;
    const uint8_t* const scales = c.matrix.scales + piece.row * c.matrix.scale_stride;
    char* const to = static_cast<char*>(c.data) + piece.row * c.rs * Bytes(kType);
    const int64_t unit0 = int64_t(piece.segment) * (64 * kUnits) + lane;
    const bool whole = (int64_t(piece.segment) + 1) * (512 * kUnits) <= cols;
    uint32_t packed[kUnits];
    int scale[kUnits];
    if (whole) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int64_t first = (unit0 + u * 64) * 8;
        scale[u] = scales[first / kBlock];
        packed[u] = *reinterpret_cast<const u32_unaligned*>(data + first / 2);
      }
    } else {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int64_t first = (unit0 + u * 64) * 8;
        packed[u] = 0;
        scale[u] = first < cols ? scales[first / kBlock] : 0;
        if (first + 8 <= cols)
          packed[u] = *reinterpret_cast<const u32_unaligned*>(data + first / 2);
        else
          for (int b = 0; b < 4; ++b)
            if (first + 2 * b < cols) packed[u] |= uint32_t(data[first / 2 + b]) << (8 * b);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int64_t first = (unit0 + u * 64) * 8;
      const float power = PowerOf(scale[u]);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = ValueOf(packed[u] >> (4 * e) & 15) * power;
      if (whole || first + 8 <= cols) {
        Unit<kType> held;
        held.Store(to, first, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (first + e < cols) StoreFloat(to, kType, first + e, v[e]);
      }
    }
  }
}

// ---- Any order and stride ----

__global__ __launch_bounds__(256) void GenericQuantizeKernel(ConvertCall c) {
  const int cols = c.matrix.cols, blocks = static_cast<int>((int64_t(cols) + kBlock - 1) / kBlock);
  const int64_t all = int64_t(c.rows) * blocks;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(gridDim.x) * 256) {
    const int block = static_cast<int>(i / c.rows), row = static_cast<int>(i - int64_t(block) * c.rows);
    const int64_t first = int64_t(block) * kBlock;
    const auto value = [&](int64_t col) { return col < cols ? LoadFloat(c.data, c.type, row * c.rs + col * c.cs) : 0.0f; };
    uint32_t largest = 0;
    for (int e = 0; e < kBlock; ++e) largest = max(largest, __float_as_uint(value(first + e)) & 0x7fffffffu);
    const int scale = ScaleOf(largest);
    const float inverse = InverseOf(scale);
    for (int e = 0; e < kBlock && first + e < cols; e += 8) {
      float v[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x] = value(first + e + x) * inverse;
      const uint32_t packed = scale == kNaNScale ? 0 : Round8(v);
      ForEachPlace(c, row, [&](int to) {
        for (int b = 0; b < 4; ++b)
          if (first + e + 2 * b < cols)
            c.matrix.data[to * c.matrix.row_bytes + (first + e) / 2 + b] = static_cast<uint8_t>(packed >> (8 * b));
      });
    }
    ForEachPlace(c, row, [&](int to) { c.matrix.scales[to * c.matrix.scale_stride + block] = static_cast<uint8_t>(scale); });
  }
}

__global__ __launch_bounds__(256) void GenericDequantizeKernel(ConvertCall c) {
  const int cols = c.matrix.cols;
  const int64_t all = int64_t(c.rows) * cols;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(gridDim.x) * 256) {
    // (Rows side by side in the destination: lanes go along them.)
    const int64_t fast = c.rs == 1 ? c.rows : cols, slow = i / fast, rest = i - slow * fast;
    const int64_t row = c.rs == 1 ? rest : slow, col = c.rs == 1 ? slow : rest;
    const uint32_t q = c.matrix.data[row * c.matrix.row_bytes + col / 2] >> (4 * (col & 1)) & 15;
    StoreFloat(c.data, c.type, row * c.rs + col * c.cs,
               ValueOf(q) * PowerOf(c.matrix.scales[row * c.matrix.scale_stride + col / kBlock]));
  }
}

unsigned BlocksFor(int64_t work, int threads) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((work + threads - 1) / threads, 1 << 20)));
}

// Segments of 64 * units units, and how many units: as many as leave every CU some waves.
template <class F>
void WithUnits(const ConvertCall& c, int compute_units, F&& f) {
  const auto segments = [&](int units) { return (int64_t(c.matrix.cols) + 512 * units - 1) / (512 * units); };
  const auto launch = [&](auto units) { f(units, int(segments(units)), BlocksFor(c.rows * segments(units), 4)); };
  if (c.rows * segments(4) >= int64_t(16) * compute_units) return launch(std::integral_constant<int, 4>());
  launch(std::integral_constant<int, 1>());
}

}  // namespace

bool LaunchQuantize(hipStream_t stream, const ConvertCall& c, int compute_units, hipError_t* status) {
  if (c.cs != 1 && c.matrix.cols != 1) return false;
  WithUnits(c, compute_units, [&](auto units, int segments, unsigned blocks) {
    constexpr int kUnits = decltype(units)::value;
    const dim3 grid(blocks), block(256);
    if (c.type == RUYAMD_DTYPE_BF16)
      hipLaunchKernelGGL((QuantizeKernel<RUYAMD_DTYPE_BF16, kUnits>), grid, block, 0, stream, c, segments);
    else if (c.type == RUYAMD_DTYPE_F16)
      hipLaunchKernelGGL((QuantizeKernel<RUYAMD_DTYPE_F16, kUnits>), grid, block, 0, stream, c, segments);
    else
      hipLaunchKernelGGL((QuantizeKernel<RUYAMD_DTYPE_F32, kUnits>), grid, block, 0, stream, c, segments);
  });
  *status = hipGetLastError();
  return true;
}

bool LaunchDequantize(hipStream_t stream, const ConvertCall& c, int compute_units, hipError_t* status) {
  if (c.cs != 1 && c.matrix.cols != 1) return false;
  WithUnits(c, compute_units, [&](auto units, int segments, unsigned blocks) {
    constexpr int kUnits = decltype(units)::value;
    const dim3 grid(blocks), block(256);
    if (c.type == RUYAMD_DTYPE_BF16)
      hipLaunchKernelGGL((DequantizeKernel<RUYAMD_DTYPE_BF16, kUnits>), grid, block, 0, stream, c, segments);
    else if (c.type == RUYAMD_DTYPE_F16)
      hipLaunchKernelGGL((DequantizeKernel<RUYAMD_DTYPE_F16, kUnits>), grid, block, 0, stream, c, segments);
    else
      hipLaunchKernelGGL((DequantizeKernel<RUYAMD_DTYPE_F32, kUnits>), grid, block, 0, stream, c, segments);
  });
  *status = hipGetLastError();
  return true;
}

hipError_t LaunchGenericQuantize(hipStream_t stream, const ConvertCall& c) {
  const int64_t blocks = (int64_t(c.matrix.cols) + kBlock - 1) / kBlock;
  hipLaunchKernelGGL(GenericQuantizeKernel, dim3(BlocksFor(c.rows * blocks, 256)), dim3(256), 0, stream, c);
  return hipGetLastError();
}
hipError_t LaunchGenericDequantize(hipStream_t stream, const ConvertCall& c) {
  hipLaunchKernelGGL(GenericDequantizeKernel, dim3(BlocksFor(int64_t(c.rows) * c.matrix.cols, 256)), dim3(256), 0, stream, c);
  return hipGetLastError();
}

}  // namespace mxfp4
}  // namespace ruyamd
