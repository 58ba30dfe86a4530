// What the kernels of grouped products share: 16-bit floating types, the
// groups' bounds, the write-back.
#ifndef RUY_AMD_CSRC_KERNELS_GROUPED_DEVICE_H_
#define RUY_AMD_CSRC_KERNELS_GROUPED_DEVICE_H_

#include <hip/hip_runtime.h>

#include "grouped.h"

namespace ruyamd {
namespace grouped {

// Value number i of a matrix of one of the three floating types.
__device__ __forceinline__ float LoadFloat(const void* p, int type, int64_t i) {
  if (type == RUYAMD_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (type == RUYAMD_DTYPE_BF16) return static_cast<float>(static_cast<const __bf16*>(p)[i]);
  return static_cast<float>(static_cast<const _Float16*>(p)[i]);
}
// (To nearest, ties to even, once.)
__device__ __forceinline__ void StoreFloat(void* p, int type, int64_t i, float v) {
  if (type == RUYAMD_DTYPE_F32)
    static_cast<float*>(p)[i] = v;
  else if (type == RUYAMD_DTYPE_BF16)
    static_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
  else
    static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
}

// Two values rounded to a 16-bit type, in one register.
template <int kType>
__device__ __forceinline__ int RoundPair(float x, float y) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f both = {x, y};
  if constexpr (kType == RUYAMD_DTYPE_BF16) {
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(int, __builtin_convertvector(both, v2bf));
  } else {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(int, __builtin_convertvector(both, v2h));
  }
}

// min first, then max, as ruy does it (ruy/reference_mul.h:47-48); a NaN stays one.
__device__ __forceinline__ float Clamp(float v, float low, float high) {
  v = high < v ? high : v;
  return v < low ? low : v;
}

// Where a group begins and ends: the caller's offsets held to 0 .. total.
struct Range {
  int begin;
  int count;
};
__device__ __forceinline__ int HeldTo(int offset, int total) { return max(0, min(offset, total)); }
__device__ __forceinline__ Range RangeOf(const int32_t* offsets, int group, int total) {
  if (!offsets) return {0, total};
  const int begin = HeldTo(offsets[group], total);
  return {begin, max(0, HeldTo(offsets[group + 1], total) - begin)};
}

}  // namespace grouped
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_GROUPED_DEVICE_H_
