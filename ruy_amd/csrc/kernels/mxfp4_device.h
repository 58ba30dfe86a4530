// Arithmetic of microscaled 4-bit floating point on the device.
#ifndef RUY_AMD_CSRC_KERNELS_MXFP4_DEVICE_H_
#define RUY_AMD_CSRC_KERNELS_MXFP4_DEVICE_H_

#include <hip/hip_runtime.h>

#include "mxfp4.h"

namespace ruyamd {
namespace mxfp4 {

constexpr int kNaNScale = 255;

// 2^(scale - 127), NaN for 255.
__device__ __forceinline__ float PowerOf(int scale) {
  const uint32_t bits = scale == kNaNScale ? 0x7fc00000u : scale == 0 ? 0x00400000u : static_cast<uint32_t>(scale) << 23;
  return __uint_as_float(bits);
}

// The scale of a block whose largest magnitude has these bits (of fp32; a NaN's are the
// largest of all): its power of two divided by 4, 2^-127 at least.
__device__ __forceinline__ int ScaleOf(uint32_t largest) {
  const int exponent = static_cast<int>(largest >> 23);
  return exponent == 255 ? kNaNScale : max(exponent - 2, 0);
}
// What the block's values are multiplied with; 0 where they are NaN (and 0 becomes of them).
__device__ __forceinline__ float InverseOf(int scale) {
  return scale == kNaNScale ? 0.0f : __uint_as_float(static_cast<uint32_t>(254 - scale) << 23);
}

// Eight values, already divided by their scales, as 4-bit numbers, the first one lowest. (The
// instruction rounds to nearest, ties to even, and gives 6 for what is larger.)
__device__ __forceinline__ uint32_t Round8(const float (&v)[8]) {
  uint32_t x = 0;
  x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(x, v[0], v[1], 1.0f, 0);
  x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(x, v[2], v[3], 1.0f, 1);
  x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(x, v[4], v[5], 1.0f, 2);
  x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(x, v[6], v[7], 1.0f, 3);
  return x;
}

// A 4-bit number's value.
__device__ __forceinline__ float ValueOf(uint32_t q) {
  const uint32_t size = q & 7;
  // 0 and 0.5 are small; above, two bits of exponent and one of mantissa.
  const float v = size < 2 ? 0.5f * size : __uint_as_float((126u << 23) + (size << 22));
  return q & 8 ? -v : v;
}

}  // namespace mxfp4
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_MXFP4_DEVICE_H_
