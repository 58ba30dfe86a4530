// Tokens to their experts and back (ruyamd_sort_tokens, ruyamd_dispatch_tokens,
// ruyamd_combine_tokens, ruyamd_combine_tokens_gradients): what the host hands to
// their kernels.
#ifndef RUY_AMD_CSRC_KERNELS_ROUTING_H_
#define RUY_AMD_CSRC_KERNELS_ROUTING_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../internal.h"

namespace ruyamd {
namespace routing {

// The choices to be sorted: number (j, t) lies at experts + j * rs + t * cs values of `wide` ? 8 : 4 bytes.
struct SortCall {
  const void* experts = nullptr;
  int64_t rs = 0, cs = 0;
  bool wide = false;
  int tokens = 0, top = 0, count = 0;
  int32_t* offsets = nullptr;
  int32_t* places = nullptr;
  int32_t* sources = nullptr;  // or null
};
hipError_t LaunchSort(hipStream_t stream, const SortCall& call, bool force_generic);

// A matrix whose element (r, c) lies at data + r * rs + c * cs values.
struct View {
  void* data = nullptr;
  int64_t rs = 0, cs = 0;
  int type = 0;
};

// One of the other calls. Places outside 0 .. columns - 1 are none.
struct Call {
  const int32_t* places = nullptr;
  int tokens = 0, top = 0;
  int width = 0;    // values of a token
  int columns = 0;  // of the matrix of places
  View token_side;  // dispatch: src; combine: dst; gradients: grad
  View place_side;  // dispatch: dst; combine, gradients: src (data may be null)
  View weights;     // data null: ones
  View grad_src, grad_weights;  // gradients only; data null: not wanted
};

// 16 bytes to a lane, where a token's values lie side by side. False: the call is not one for
// these, and nothing was launched.
bool LaunchDispatch(hipStream_t stream, const Call& call, int compute_units, hipError_t* status);
bool LaunchCombine(hipStream_t stream, const Call& call, int compute_units, hipError_t* status);
bool LaunchGradients(hipStream_t stream, const Call& call, int compute_units, hipError_t* status);

// One value to a lane; any order and stride.
hipError_t LaunchGenericDispatch(hipStream_t stream, const Call& call);
hipError_t LaunchGenericCombine(hipStream_t stream, const Call& call);
hipError_t LaunchGenericGradients(hipStream_t stream, const Call& call);

}  // namespace routing
}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_KERNELS_ROUTING_H_
