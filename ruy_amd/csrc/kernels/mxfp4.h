// Microscaled 4-bit floating point (ruyamd_quantize_mxfp4, ruyamd_dequantize_mxfp4,
// ruyamd_mul_mxfp4): what the host hands to their kernels.
#ifndef RUY_AMD_CSRC_KERNELS_MXFP4_H_
#define RUY_AMD_CSRC_KERNELS_MXFP4_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../internal.h"

namespace ruyamd {
namespace mxfp4 {

constexpr int kBlock = 32;  // values to a scale, 16 bytes

// Rows of 4-bit values and their scales.
struct Matrix {
  uint8_t* data = nullptr;
  uint8_t* scales = nullptr;
  int rows = 0, cols = 0;
  int64_t row_bytes = 0, scale_stride = 0, matrix_bytes = 0, scales_matrix_stride = 0;
};

// To or from 4 bits: element (r, c) of the other side lies at data + r * rs + c * cs values.
struct ConvertCall {
  void* data = nullptr;
  int64_t rs = 0, cs = 0;
  int type = 0;
  int rows = 0;  // of the other side
  Matrix matrix;
  // Rows go to these places (top to a row) where there are any.
  const int32_t* places = nullptr;
  int top = 0;
};
// 8 values to a lane, where a row's lie side by side. False: not one for these, and nothing was launched.
bool LaunchQuantize(hipStream_t stream, const ConvertCall& call, int compute_units, hipError_t* status);
bool LaunchDequantize(hipStream_t stream, const ConvertCall& call, int compute_units, hipError_t* status);
// One block to a lane; one value to a lane.
hipError_t LaunchGenericQuantize(hipStream_t stream, const ConvertCall& call);
hipError_t LaunchGenericDequantize(hipStream_t stream, const ConvertCall& call);

// A product: dst element (i, j) lies at dst + i * dst_rs + j * dst_cs.
struct MulCall {
  Matrix lhs, rhs;  // rhs: a row to each column of dst
  void* dst = nullptr;
  int64_t dst_rs = 0, dst_cs = 0;
  int dst_type = 0;
  int m = 0, n = 0, k = 0;
  const int32_t* offsets = nullptr;  // null: one group that has all columns
  int groups = 1;
  const float* bias = nullptr;
  int64_t bias_stride = 0;
  float clamp_min = 0, clamp_max = 0;
  int compute_units = 0;
  int forced_tile_rows = 0, forced_tile_cols = 0;  // 0: the fastest one
  bool forced_deep = false;                        // of 64x64 and 128x128, those with four stages
};
// As in grouped.h.
hipError_t LaunchGeneric(hipStream_t stream, const MulCall& call);
bool LaunchTiles(hipStream_t stream, const MulCall& call, hipError_t* status);
float TilesMicroseconds(const MulCall& call);  // how long that takes, about; negative: not a call for them
// (Also where tiles would take less time.)
bool LaunchStream(hipStream_t stream, const MulCall& call, hipError_t* status);

}  // namespace mxfp4
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_MXFP4_H_
