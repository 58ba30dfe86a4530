// Products of two matrices of microscaled 4-bit values, one destination element to a lane: the
// kernel that takes every size and stride, and that the others are tested against. A
// block's sum is exact; the sum over blocks is fp32, in ascending order of the depth. Arithmetic of a value at a time bounds it: 8192 x 8192 x
// 8192 takes 987 ms, four thousand times as long as on the matrix cores; calls that come here have depths below 32, or sizes that no
// other kernel's offsets or grid reach.
#include "grouped_device.h"
#include "launch_geometry.h"
#include "mxfp4_device.h"

namespace ruyamd {
namespace mxfp4 {
namespace {

using grouped::Clamp;
using grouped::Range;
using grouped::RangeOf;
using grouped::StoreFloat;

constexpr int kTile = kGenericTile;

__global__ __launch_bounds__(kTile* kTile) void GenericMxFp4Kernel(MulCall c) {
  for (int g = blockIdx.z; g < c.groups; g += gridDim.z) {
    const Range range = RangeOf(c.offsets, g, c.n);
    const int64_t i = int64_t(blockIdx.x) * kTile + threadIdx.x;
    if (i >= c.m) return;
    const uint8_t* const a = c.lhs.data + g * c.lhs.matrix_bytes + i * c.lhs.row_bytes;
    const uint8_t* const a_scales = c.lhs.scales + g * c.lhs.scales_matrix_stride + i * c.lhs.scale_stride;
    for (int64_t j = int64_t(blockIdx.y) * kTile + threadIdx.y; j < range.count; j += int64_t(gridDim.y) * kTile) {
      const int64_t column = range.begin + j;
      const uint8_t* const b = c.rhs.data + column * c.rhs.row_bytes;
      const uint8_t* const b_scales = c.rhs.scales + column * c.rhs.scale_stride;
      float sum = 0;
      for (int64_t k0 = 0; k0 < c.k; k0 += kBlock) {
        float block = 0;
        for (int64_t k = k0; k < min(k0 + kBlock, int64_t(c.k)); ++k)
          block += ValueOf(a[k / 2] >> (4 * (k & 1)) & 15) * ValueOf(b[k / 2] >> (4 * (k & 1)) & 15);
        const int sa = a_scales[k0 / kBlock], sb = b_scales[k0 / kBlock];
        sum += sa == kNaNScale || sb == kNaNScale ? __uint_as_float(0x7fc00000u) : ldexpf(block, sa + sb - 254);
      }
      if (c.bias) sum += c.bias[g * c.bias_stride + i];
      StoreFloat(c.dst, c.dst_type, i * c.dst_rs + column * c.dst_cs, Clamp(sum, c.clamp_min, c.clamp_max));
    }
  }
}

}  // namespace

hipError_t LaunchGeneric(hipStream_t stream, const MulCall& c) {
  const unsigned rows = static_cast<unsigned>((int64_t(c.m) + kTile - 1) / kTile);
  // (Enough of a group's columns side by side, whatever it has; the rest in turn.)
  const unsigned y = static_cast<unsigned>(min((int64_t(c.n) / c.groups + kTile) / kTile, int64_t(1024)));
  hipLaunchKernelGGL(GenericMxFp4Kernel, dim3(rows, y, static_cast<unsigned>(min(c.groups, 1024))), dim3(kTile, kTile), 0, stream, c);
  return hipGetLastError();
}

}  // namespace mxfp4
}  // namespace ruyamd
