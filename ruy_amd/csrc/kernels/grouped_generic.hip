// Grouped and 4-bit products, one destination element to a lane: the kernel
// that takes every type, order, stride and alignment, and that the others are
// tested against. Its sums are fp32, in ascending order of the depth.
#include "grouped_device.h"
#include "launch_geometry.h"

namespace ruyamd {
namespace grouped {
namespace {

constexpr int kTile = kGenericTile;

// grid.z walks the groups; x and y the rows and columns of one, y with a stride
// (how many columns a group has is known here only).
template <bool kInt4>
__global__ __launch_bounds__(kTile* kTile) void GenericGroupedKernel(Call c, Int4 w) {
  for (int g = blockIdx.z; g < c.groups; g += gridDim.z) {
    const bool by_columns = c.dealt == Dealt::kColumns;
    const Range range = RangeOf(c.offsets, g, by_columns ? c.n : c.k);
    const int64_t i = int64_t(blockIdx.x) * kTile + threadIdx.x;
    if (i >= c.m) return;
    const int columns = by_columns ? range.count : c.n;
    const int depth = by_columns ? c.k : range.count;
    const int64_t first_column = by_columns ? range.begin : 0;
    const int64_t first_depth = by_columns ? 0 : range.begin;
    const int64_t lhs_at = i * c.lhs_rs + first_depth * c.lhs_cs + (by_columns ? g * c.matrix_stride : 0);
    const int64_t dst_at = by_columns ? 0 : g * c.matrix_stride;
    for (int64_t j = int64_t(blockIdx.y) * kTile + threadIdx.y; j < columns; j += int64_t(gridDim.y) * kTile) {
      const int64_t rhs_at = (first_column + j) * c.rhs_cs + first_depth * c.rhs_rs;
      float sum = 0;
      for (int k = 0; k < depth; ++k) {
        const float r = LoadFloat(c.rhs, c.type, rhs_at + k * c.rhs_rs);
        float l;
        if constexpr (kInt4) {
          const uint8_t pair = w.data[g * w.matrix_bytes + i * w.row_bytes + k / 2];
          const int64_t at = g * w.scales_matrix_stride + i * w.scale_stride + k / w.group_size;
          const int q = k & 1 ? pair >> 4 : pair & 15;
          const int zero = w.zero_points ? w.zero_points[at] : 8;
          l = static_cast<float>(q - zero) * LoadFloat(w.scales, w.scale_type, at);
        } else {
          l = LoadFloat(c.lhs, c.type, lhs_at + k * c.lhs_cs);
        }
        sum += l * r;
      }
      if (c.bias) sum += c.bias[g * c.bias_stride + i];
      StoreFloat(c.dst, c.dst_type, dst_at + i * c.dst_rs + (first_column + j) * c.dst_cs,
                 Clamp(sum, c.clamp_min, c.clamp_max));
    }
  }
}

}  // namespace

hipError_t LaunchGeneric(hipStream_t stream, const Call& call, const Int4* weights) {
  const unsigned rows = static_cast<unsigned>((int64_t(call.m) + kTile - 1) / kTile);
  // (Enough of a group's columns side by side, whatever it has; the rest in turn.)
  const int64_t columns = call.dealt == Dealt::kColumns ? call.n / call.groups + 1 : call.n;
  const unsigned y = static_cast<unsigned>(min((columns + kTile - 1) / kTile, int64_t(1024)));
  const dim3 grid(rows, y, static_cast<unsigned>(min(call.groups, 1024))), block(kTile, kTile);
  if (weights)
    hipLaunchKernelGGL(GenericGroupedKernel<true>, grid, block, 0, stream, call, *weights);
  else
    hipLaunchKernelGGL(GenericGroupedKernel<false>, grid, block, 0, stream, call, Int4{});
  return hipGetLastError();
}

}  // namespace grouped
}  // namespace ruyamd
