// The 256x256 tile of products of 4-bit values (mxfp4_large.hip).
#ifndef RUY_AMD_CSRC_KERNELS_MXFP4_LARGE_H_
#define RUY_AMD_CSRC_KERNELS_MXFP4_LARGE_H_

#include "mxfp4.h"

namespace ruyamd {
namespace mxfp4 {

// The largest tiles. Operands straight to LDS: rows of data and of scales begin at multiples of 4 bytes, the depth is a multiple of
// 128 (16 bytes of scales then end at a multiple of 4) and 512 at least (a row has 16).
hipError_t LaunchLarge(hipStream_t stream, const MulCall& call, unsigned blocks);  // 256x256
hipError_t LaunchWide(hipStream_t stream, const MulCall& call, unsigned blocks);   // 256x128

}  // namespace mxfp4
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_MXFP4_LARGE_H_
