// The streaming kernels of 4-bit weights for tokens of one type.
#include "grouped_stream.h"

namespace ruyamd {
namespace grouped {

hipError_t LaunchStreamInt4F32(hipStream_t stream, const StreamArgs& args, const StreamPlan& plan) {
  return LaunchStreamInt4<RUYAMD_DTYPE_F32>(stream, args, plan);
}

}  // namespace grouped
}  // namespace ruyamd
