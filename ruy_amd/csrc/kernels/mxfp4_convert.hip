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
  // Where the row ends `left` values behind `row` (maybe inside the unit, or in front of it): zeros behind. (It has 16 bytes; all lanes
  // load at once, which those that end the row would not if they took its last values one by one.)
  __device__ __forceinline__ void LoadEnd(const char* row, int first, int left) {
#pragma unroll
    for (int i = 0; i < kGranules; ++i)
      raw[i] = granule::LoadGranule<false>(reinterpret_cast<const uint8_t*>(row), first * Bytes(kType) + i * 16, left * Bytes(kType));
#pragma unroll
    for (int i = 0; i < kGranules; ++i) raw[i] = granule::PlaceGranule(raw[i], first * Bytes(kType) + i * 16, left * Bytes(kType));
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
    if (whole) {
      Unit<kType> held[kUnits];
#pragma unroll
      for (int u = 0; u < kUnits; ++u) held[u].Load(from, (unit0 + u * 64) * 8);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) held[u].Values(v[u]);
    } else {
      const int64_t segment = int64_t(piece.segment) * (512 * kUnits);
      Unit<kType> held[kUnits];
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        held[u].LoadEnd(from + segment * Bytes(kType), (u * 64 + lane) * 8, static_cast<int>(cols - segment));
#pragma unroll
      for (int u = 0; u < kUnits; ++u) held[u].Values(v[u]);
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

// ---- Rows of 256 values or less ----
//
// kLanes lanes have a row, a unit of 8 values each: 64 / kLanes rows to a wave. (100000 x 128 bfloat16 values, a wave to a row and so: 57 and 8 us,
// back 72 and 8.6.)

template <int kType, int kLanes>
__global__ __launch_bounds__(256) void NarrowQuantizeKernel(ConvertCall c) {
  const int cols = c.matrix.cols, mine = threadIdx.x & (kLanes - 1), first = mine * 8;
  for (int64_t row0 = int64_t(blockIdx.x) * (256 / kLanes); row0 < c.rows; row0 += int64_t(gridDim.x) * (256 / kLanes)) {
    const int64_t row = row0 + threadIdx.x / kLanes;
    const bool there = row < c.rows && first < cols;  // (all lanes go through the exchanges)
    const char* const from = static_cast<const char*>(c.data) + row * c.rs * Bytes(kType);
    float v[8] = {};
    if (there && cols * Bytes(kType) >= 16) {
      Unit<kType> held;
      held.LoadEnd(from, first, cols);
      held.Values(v);
    } else if (there) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (first + e < cols) v[e] = LoadFloat(from, kType, first + e);
    }
    uint32_t largest = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) largest = max(largest, __float_as_uint(v[e]) & 0x7fffffffu);
    const int scale = ScaleOf(LargestOfFour(largest));
    const float inverse = InverseOf(scale);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= inverse;
    const uint32_t packed = scale == kNaNScale ? 0 : Round8(v);
    if (!there) continue;
    ForEachPlace(c, static_cast<int>(row), [&](int to) __attribute__((always_inline)) {
      uint8_t* const data = c.matrix.data + to * c.matrix.row_bytes;
      if ((mine & 3) == 0) c.matrix.scales[to * c.matrix.scale_stride + first / kBlock] = static_cast<uint8_t>(scale);
      if (first + 8 <= cols) {
        *reinterpret_cast<u32_unaligned*>(data + first / 2) = packed;
      } else {
        for (int b = 0; b < (cols - first + 1) / 2; ++b) data[first / 2 + b] = static_cast<uint8_t>(packed >> (8 * b));
      }
    });
  }
}

template <int kType, int kLanes>
__global__ __launch_bounds__(256) void NarrowDequantizeKernel(ConvertCall c) {
  const int cols = c.matrix.cols, first = (threadIdx.x & (kLanes - 1)) * 8;
  if (first >= cols) return;
  for (int64_t row = (int64_t(blockIdx.x) * 256 + threadIdx.x) / kLanes; row < c.rows; row += int64_t(gridDim.x) * (256 / kLanes)) {
    const uint8_t* const data = c.matrix.data + row * c.matrix.row_bytes;
    char* const to = static_cast<char*>(c.data) + row * c.rs * Bytes(kType);
    const float power = PowerOf(c.matrix.scales[row * c.matrix.scale_stride + first / kBlock]);
    uint32_t packed = 0;
    if (first + 8 <= cols) {
      packed = *reinterpret_cast<const u32_unaligned*>(data + first / 2);
    } else {
      for (int b = 0; b < 4; ++b)
        if (first + 2 * b < cols) packed |= uint32_t(data[first / 2 + b]) << (8 * b);
    }
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ValueOf(packed >> (4 * e) & 15) * power;
    if (first + 8 <= cols) {
      Unit<kType> held;
      held.Store(to, first, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (first + e < cols) StoreFloat(to, kType, first + e, v[e]);
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

// Segments of 64 * units units, and how many units: no more than a row has, and as many as leave every CU some waves.
template <class F>
void WithUnits(const ConvertCall& c, int compute_units, F&& f) {
  const auto segments = [&](int units) { return (int64_t(c.matrix.cols) + 512 * units - 1) / (512 * units); };
  const auto launch = [&](auto units) { f(units, int(segments(units)), BlocksFor(c.rows * segments(units), 4)); };
  const int64_t enough = int64_t(16) * compute_units;
  if (c.matrix.cols > 1024 && c.rows * segments(4) >= enough) return launch(std::integral_constant<int, 4>());
  if (c.matrix.cols > 512 && c.rows * segments(2) >= enough) return launch(std::integral_constant<int, 2>());
  launch(std::integral_constant<int, 1>());
}
// Lanes to a narrow row: f(lanes as a constant, blocks), or false for one that is not narrow.
template <class F>
bool WithLanes(const ConvertCall& c, F&& f) {
  const auto launch = [&](auto lanes) { f(lanes, BlocksFor(int64_t(c.rows) * decltype(lanes)::value, 256)); };
  if (c.matrix.cols > 256) return false;
  if (c.matrix.cols > 128)
    launch(std::integral_constant<int, 32>());
  else if (c.matrix.cols > 64)
    launch(std::integral_constant<int, 16>());
  else
    launch(std::integral_constant<int, 8>());
  return true;
}
// f(type as a constant).
template <class F>
void WithType(int type, F&& f) {
  if (type == RUYAMD_DTYPE_BF16) return f(std::integral_constant<int, RUYAMD_DTYPE_BF16>());
  if (type == RUYAMD_DTYPE_F16) return f(std::integral_constant<int, RUYAMD_DTYPE_F16>());
  f(std::integral_constant<int, RUYAMD_DTYPE_F32>());
}

}  // namespace

bool LaunchQuantize(hipStream_t stream, const ConvertCall& c, int compute_units, hipError_t* status) {
  if (c.cs != 1 && c.matrix.cols != 1) return false;
  WithType(c.type, [&](auto type) {
    constexpr int kType = decltype(type)::value;
    const bool narrow = WithLanes(c, [&](auto lanes, unsigned blocks) {
      hipLaunchKernelGGL((NarrowQuantizeKernel<kType, decltype(lanes)::value>), dim3(blocks), dim3(256), 0, stream, c);
    });
    if (!narrow) WithUnits(c, compute_units, [&](auto units, int segments, unsigned blocks) {
      hipLaunchKernelGGL((QuantizeKernel<kType, decltype(units)::value>), dim3(blocks), dim3(256), 0, stream, c, segments);
    });
  });
  *status = hipGetLastError();
  return true;
}

bool LaunchDequantize(hipStream_t stream, const ConvertCall& c, int compute_units, hipError_t* status) {
  if (c.cs != 1 && c.matrix.cols != 1) return false;
  WithType(c.type, [&](auto type) {
    constexpr int kType = decltype(type)::value;
    const bool narrow = WithLanes(c, [&](auto lanes, unsigned blocks) {
      hipLaunchKernelGGL((NarrowDequantizeKernel<kType, decltype(lanes)::value>), dim3(blocks), dim3(256), 0, stream, c);
    });
    if (!narrow) WithUnits(c, compute_units, [&](auto units, int segments, unsigned blocks) {
      hipLaunchKernelGGL((DequantizeKernel<kType, decltype(units)::value>), dim3(blocks), dim3(256), 0, stream, c, segments);
    });
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
