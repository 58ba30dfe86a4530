// Arithmetic of microscaled 4-bit floating point on the device.
#ifndef RUY_AMD_CSRC_KERNELS_MXFP4_DEVICE_H_
#define RUY_AMD_CSRC_KERNELS_MXFP4_DEVICE_H_

#include <hip/hip_runtime.h>

#include "granule.h"
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

// ---- For the matrix instructions ----
//
// v_mfma_scale_f32_16x16x128 takes 16 bytes of 4-bit values from each lane: lane l has row (column) l % 16
// and the block number l / 16 of four. The power of two of the lane's block is one byte of a register, and
// which byte is part of the instruction. So 16 blocks of a row, 512 values, are four instructions with block 4 i + l / 16
// in the i-th; the scales that lane l needs for them, bytes l / 16, 4 + l / 16, .. of the row's 16, are one word of these
// 16 bytes transposed.
constexpr int kChunk = 16 * kBlock;  // depth positions to a transposition

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
using granule::v4i;

// acc += a b of 16 rows by 16 columns and 128 values of depth, with byte kByte of either side's scales.
template <int kByte>
__device__ __forceinline__ void Mma(const v4i& a, const v4i& b, int a_scales, int b_scales, v4f& acc) {
  const v8i a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  constexpr int kE2M1 = 4;
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, acc, kE2M1, kE2M1, kByte, a_scales, kByte, b_scales);
}

// Four words of four bytes, transposed.
__device__ __forceinline__ v4i Transposed(const v4i& x) {
  const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400), b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602);
  const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602);
  return v4i{static_cast<int>(__builtin_amdgcn_perm(c, a, 0x05040100)), static_cast<int>(__builtin_amdgcn_perm(c, a, 0x07060302)),
             static_cast<int>(__builtin_amdgcn_perm(d, b, 0x05040100)), static_cast<int>(__builtin_amdgcn_perm(d, b, 0x07060302))};
}
// Word q of the transposition alone; `selector`: ColumnSelector(q).
__device__ __forceinline__ uint32_t ColumnSelector(int q) { return static_cast<uint32_t>(q | (q + 4) << 8); }
__device__ __forceinline__ int ColumnOf(const v4i& x, uint32_t selector) {
  const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], selector), b = __builtin_amdgcn_perm(x[3], x[2], selector);
  return static_cast<int>(__builtin_amdgcn_perm(b, a, 0x05040100));
}

// A row's scales number `first` .. first + 15 of `count`, zeros (which are no NaN) behind the last. The load and what
// makes that of it, apart.
__device__ __forceinline__ v4i LoadScales(const uint8_t* row, int first, int count) {
  return count >= 16 ? granule::LoadGranule<false>(row, first, count) : granule::LoadGranule<true>(row, first, count);
}
__device__ __forceinline__ v4i PlaceScales(const v4i& x, int first, int count) {
  return count >= 16 ? granule::PlaceGranule<false>(x, first, count) : granule::PlaceGranule<true>(x, first, count);
}

// 16 bytes of values from depth position k on, of which `depth` are the row's: zeros behind. (For those that have been
// moved to their place: the unused half of an odd row's last byte is cleared.)
__device__ __forceinline__ v4i WithoutOddHalf(v4i x, int64_t k, int64_t depth) {
  const int64_t last = depth - k;  // odd, 1 .. 31: the value's number whose half is to be cleared
  if (last > 0 && last < kBlock && (last & 1)) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (last / 8 == e) x[e] &= static_cast<int>(~(0xf0u << (static_cast<int>(last) % 8 / 2 * 8)));
  }
  return x;
}

}  // namespace mxfp4
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_MXFP4_DEVICE_H_
