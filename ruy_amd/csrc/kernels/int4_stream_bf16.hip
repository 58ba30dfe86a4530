// The streaming kernels of 4-bit weights for tokens of one type.
#include "grouped_stream.h"

namespace ruyamd {
namespace grouped {

hipError_t LaunchStreamInt4Bf16(hipStream_t stream, const StreamArgs& args, unsigned blocks, int waves, int rows, int cols) {
  return LaunchStreamType<true, RUYAMD_DTYPE_BF16>(stream, args, blocks, waves, rows, cols);
}

}  // namespace grouped
}  // namespace ruyamd
