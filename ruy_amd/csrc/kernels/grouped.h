// Products whose columns or depth are dealt to groups (ruyamd_mul_grouped,
// ruyamd_mul_grouped_depth) and products with 4-bit weights (ruyamd_mul_int4):
// what the host hands to their kernels.
#ifndef RUY_AMD_CSRC_KERNELS_GROUPED_H_
#define RUY_AMD_CSRC_KERNELS_GROUPED_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../internal.h"

namespace ruyamd {
namespace grouped {

// The dimension that is dealt to groups.
enum class Dealt { kColumns, kDepth };

// One call. Strides are in values; element (r, c) of a matrix lies at
// data + r * rs + c * cs, and one of rs and cs is 1.
struct Call {
  Dealt dealt = Dealt::kColumns;
  const void* lhs = nullptr;  // of the first group (kColumns)
  const void* rhs = nullptr;
  void* dst = nullptr;        // of the first group (kDepth)
  int64_t lhs_rs = 0, lhs_cs = 0, rhs_rs = 0, rhs_cs = 0, dst_rs = 0, dst_cs = 0;
  int64_t matrix_stride = 0;
  // (No offsets: one group that has all columns.)
  const int32_t* offsets = nullptr;
  int groups = 1;
  int m = 0, n = 0, k = 0;    // n (k) is the sum over all groups
  int type = 0, dst_type = 0;
  const float* bias = nullptr;
  int64_t bias_stride = 0;
  float clamp_min = 0, clamp_max = 0;
  int compute_units = 0;
  int forced_tile_rows = 0, forced_tile_cols = 0;  // 0: the fastest one
};

// The 4-bit left-hand operand of a call (lhs, lhs_rs and lhs_cs of which are unused).
struct Int4 {
  const uint8_t* data = nullptr;
  const void* scales = nullptr;
  const uint8_t* zero_points = nullptr;
  int group_size = 0;  // depth positions to a scale
  int scale_type = 0;
  int64_t row_bytes = 0, scale_stride = 0, matrix_bytes = 0, scales_matrix_stride = 0;
};

// One destination element to a lane; takes every call. (The other kernels are
// tested against it, and it takes what they do not.)
hipError_t LaunchGeneric(hipStream_t stream, const Call& call, const Int4* weights);

// Tiles of the destination on the matrix cores (grouped_gemm.h). False: the call is
// not one for this kernel, and nothing was launched.
bool LaunchTiles(hipStream_t stream, const Call& call, hipError_t* status);

// Every weight read once (grouped_stream.h): 4-bit weights, and others by rows against a
// few columns a group. False as above.
bool LaunchStream(hipStream_t stream, const Call& call, const Int4* weights, hipError_t* status);

}  // namespace grouped
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_GROUPED_H_
