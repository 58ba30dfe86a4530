#include "checks.h"

#include <cmath>

namespace ruyamd {

int Fail(ruyamd_ctx* ctx, int code, const std::string& msg) {
  ctx->last_error = msg;
  return code;
}

bool IsOperandType(int dtype) {
  return dtype == RUYAMD_DTYPE_F32 || dtype == RUYAMD_DTYPE_BF16 || dtype == RUYAMD_DTYPE_F16;
}

int CheckMatrix(ruyamd_ctx* ctx, const ruyamd_mat& m, const std::string& name) {
  if (m.rows < 0 || m.cols < 0) return Fail(ctx, RUYAMD_E_INVALID, name + ": negative size");
  if (m.order != RUYAMD_ORDER_COL_MAJOR && m.order != RUYAMD_ORDER_ROW_MAJOR)
    return Fail(ctx, RUYAMD_E_INVALID, name + ": bad order");
  if (m.stride < (m.order == RUYAMD_ORDER_COL_MAJOR ? m.rows : m.cols))
    return Fail(ctx, RUYAMD_E_INVALID, name + ": stride smaller than the contiguous dimension");
  if (!IsOperandType(m.dtype)) return Fail(ctx, RUYAMD_E_UNSUPPORTED, name + ": the type must be fp32, bfloat16 or half");
  if (m.zero_point) return Fail(ctx, RUYAMD_E_INVALID, name + ": floating-point matrices need zero_point == 0");
  if (m.rows > 0 && m.cols > 0) {
    if (!m.data) return Fail(ctx, RUYAMD_E_INVALID, name + ": null data");
    const uintptr_t size = m.dtype == RUYAMD_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(m.data) % size)
      return Fail(ctx, RUYAMD_E_INVALID, name + ": data not aligned to its type");
    if (MemoryOf(m.data) != Memory::kDevice) return Fail(ctx, RUYAMD_E_UNSUPPORTED, name + ": not device memory");
  }
  return RUYAMD_OK;
}

int CheckDeviceBuffer(ruyamd_ctx* ctx, const void* p, uintptr_t alignment, const char* name) {
  if (!p) return Fail(ctx, RUYAMD_E_INVALID, std::string(name) + ": null");
  if (reinterpret_cast<uintptr_t>(p) % alignment)
    return Fail(ctx, RUYAMD_E_INVALID, std::string(name) + ": not aligned to its type");
  if (MemoryOf(p) != Memory::kDevice) return Fail(ctx, RUYAMD_E_UNSUPPORTED, std::string(name) + ": not device memory");
  return RUYAMD_OK;
}

int CheckGroups(ruyamd_ctx* ctx, const ruyamd_groups& g) {
  if (g.count < 1 || g.count > kMostGroups) return Fail(ctx, RUYAMD_E_INVALID, "groups: count must be 1 .. 65536");
  if (g.matrix_stride < 0 || g.bias_stride < 0) return Fail(ctx, RUYAMD_E_INVALID, "groups: negative stride");
  return CheckDeviceBuffer(ctx, g.offsets, 4, "groups: offsets");
}

int CheckParams(ruyamd_ctx* ctx, const ruyamd_mul_params& p, bool may_have_bias) {
  if (p.accum_dtype != RUYAMD_DTYPE_F32) return Fail(ctx, RUYAMD_E_UNSUPPORTED, "the accumulator must be fp32");
  if (p.multiplier_fixedpoint_perchannel || p.multiplier_exponent_perchannel || p.multiplier_fixedpoint ||
      p.multiplier_exponent)
    return Fail(ctx, RUYAMD_E_INVALID, "multiplier set on a floating-point product");
  if (std::isnan(p.clamp_min) || std::isnan(p.clamp_max)) return Fail(ctx, RUYAMD_E_INVALID, "clamp bounds are not numbers");
  if (p.channel_dimension > RUYAMD_CHANNEL_COL) return Fail(ctx, RUYAMD_E_INVALID, "bad channel dimension");
  if (!p.bias) return RUYAMD_OK;
  if (!may_have_bias) return Fail(ctx, RUYAMD_E_UNSUPPORTED, "ruyamd_mul_grouped_depth takes no bias");
  if (p.channel_dimension != RUYAMD_CHANNEL_ROW) return Fail(ctx, RUYAMD_E_UNSUPPORTED, "the bias must be one to each row");
  return CheckDeviceBuffer(ctx, p.bias, 4, "bias");
}

int BeginLaunch(ruyamd_ctx* ctx) {
  const int enabled = ruyamd_ctx_get_runtime_enabled_paths(ctx);
  if (!(enabled & RUYAMD_PATH_GFX950)) {
    ctx->last_used_path = RUYAMD_PATH_NONE;
    return Fail(ctx, RUYAMD_E_NO_PATH, "runtime-enabled paths exclude gfx950 and this library has no CPU path");
  }
  ctx->last_used_path = RUYAMD_PATH_GFX950;
  ctx->last_kernel = RUYAMD_KERNEL_NONE;
  int current_device = -1;
  if (hipGetDevice(&current_device) != hipSuccess || current_device != ctx->device) {
    if (hipSetDevice(ctx->device) != hipSuccess) return Fail(ctx, RUYAMD_E_HIP, "hipSetDevice failed");
  }
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(ctx->stream, &status) != hipSuccess) {
    (void)hipGetLastError();
    status = hipStreamCaptureStatusNone;
  }
  ctx->capturing = status == hipStreamCaptureStatusActive;
  return RUYAMD_OK;
}

int EndLaunch(ruyamd_ctx* ctx, bool timed, hipError_t launched) {
  if (timed) ctx->TimingEnd();
  const bool wait = ctx->synchronous && !ctx->capturing;
  ctx->capturing = false;
  if (launched != hipSuccess)
    return Fail(ctx, RUYAMD_E_HIP, std::string("kernel launch failed: ") + hipGetErrorString(launched));
  if (wait && hipStreamSynchronize(ctx->stream) != hipSuccess)
    return Fail(ctx, RUYAMD_E_HIP, std::string("kernel execution failed: ") + hipGetErrorString(hipGetLastError()));
  return RUYAMD_OK;
}

}  // namespace ruyamd
