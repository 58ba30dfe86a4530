// What the entry points for layers of experts share: the checks of their
// arguments and the launch of what was checked.
#ifndef RUY_AMD_CSRC_CHECKS_H_
#define RUY_AMD_CSRC_CHECKS_H_

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "context.h"
#include "internal.h"

namespace ruyamd {

constexpr int kMostGroups = 65536;

// The code, with the message left in the context.
int Fail(ruyamd_ctx* ctx, int code, const std::string& msg);

bool IsOperandType(int dtype);  // fp32, bfloat16, half

// A matrix of one of these types in device memory.
int CheckMatrix(ruyamd_ctx* ctx, const ruyamd_mat& m, const std::string& name);
int CheckDeviceBuffer(ruyamd_ctx* ctx, const void* p, uintptr_t alignment, const char* name);
int CheckGroups(ruyamd_ctx* ctx, const ruyamd_groups& g);
int CheckRouting(ruyamd_ctx* ctx, const ruyamd_routing& r);  // sizes and places
int CheckParams(ruyamd_ctx* ctx, const ruyamd_mul_params& p, bool may_have_bias);

// What comes before a launch on the context's stream (the path, the device, whether a graph is recorded)
// and after it: unless the context is asynchronous or its stream records a graph, the call waits.
int BeginLaunch(ruyamd_ctx* ctx);
int EndLaunch(ruyamd_ctx* ctx, bool timed, hipError_t launched);

// `launch` enqueues the kernels of a checked call, sets ctx->last_kernel and returns their status.
// nothing: the call has nothing to do.
template <class F>
int LaunchChecked(ruyamd_ctx* ctx, bool nothing, F&& launch) {
  if (int rc = BeginLaunch(ctx)) return rc;
  if (nothing) {
    ctx->capturing = false;
    return RUYAMD_OK;
  }
  const bool timed = ctx->TimingBegin();
  return EndLaunch(ctx, timed, launch());
}

}  // namespace ruyamd

#endif  // RUY_AMD_CSRC_CHECKS_H_
