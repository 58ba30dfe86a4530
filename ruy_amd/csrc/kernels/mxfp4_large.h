// The 256x256 tile of products of 4-bit values (mxfp4_large.hip).
#ifndef RUY_AMD_CSRC_KERNELS_MXFP4_LARGE_H_
#define RUY_AMD_CSRC_KERNELS_MXFP4_LARGE_H_

#include "mxfp4.h"

namespace ruyamd {
namespace mxfp4 {

// The largest tiles. Operands straight to LDS: rows of data begin at multiples of 4 bytes, the depth is a whole number of blocks, and
// 512 at least (a row has 16 scales).
// Of scales see ScaleRows (mxfp4_tile.h).
inline bool ScalesNeedWords(const MulCall& call) {
  const auto aligned = [](const Matrix& m) { return reinterpret_cast<uintptr_t>(m.scales) % 4 == 0 && m.scale_stride % 4 == 0; };
  return call.k % 128 != 0 || !aligned(call.lhs) || !aligned(call.rhs) || call.lhs.scales_matrix_stride % 4 != 0;
}
hipError_t LaunchLarge(hipStream_t stream, const MulCall& call, unsigned blocks);  // 256x256
hipError_t LaunchWide(hipStream_t stream, const MulCall& call, unsigned blocks);   // 256x128

}  // namespace mxfp4
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_MXFP4_LARGE_H_
