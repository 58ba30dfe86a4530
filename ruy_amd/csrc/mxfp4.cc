// ruyamd_quantize_mxfp4, ruyamd_dequantize_mxfp4 and ruyamd_mul_mxfp4: the checks
// of a call, the choice of its kernel, and its launch on the context's stream.
#include "kernels/mxfp4.h"

#include <string>

#include "checks.h"
#include "context.h"
#include "internal.h"

namespace ruyamd {
namespace {

// A matrix in 4 bits, its strides filled in.
int CheckMxFp4(ruyamd_ctx* ctx, const ruyamd_mxfp4_mat& m, const std::string& name, mxfp4::Matrix* out) {
  if (m.rows < 0 || m.cols < 0) return Fail(ctx, RUYAMD_E_INVALID, name + ": negative size");
  if (m.row_bytes < 0 || m.scale_stride < 0 || m.matrix_bytes < 0 || m.scales_matrix_stride < 0)
    return Fail(ctx, RUYAMD_E_INVALID, name + ": negative stride");
  const int64_t bytes = (int64_t(m.cols) + 1) / 2, scales = (int64_t(m.cols) + mxfp4::kBlock - 1) / mxfp4::kBlock;
  out->data = static_cast<uint8_t*>(m.data);
  out->scales = m.scales;
  out->rows = m.rows;
  out->cols = m.cols;
  out->row_bytes = m.row_bytes ? m.row_bytes : bytes;
  out->scale_stride = m.scale_stride ? m.scale_stride : scales;
  if (out->row_bytes < bytes || out->scale_stride < scales)
    return Fail(ctx, RUYAMD_E_INVALID, name + ": stride smaller than a row");
  out->matrix_bytes = m.matrix_bytes ? m.matrix_bytes : out->row_bytes * m.rows;
  out->scales_matrix_stride = m.scales_matrix_stride ? m.scales_matrix_stride : out->scale_stride * m.rows;
  if (m.rows > 0 && m.cols > 0) {
    if (int rc = CheckDeviceBuffer(ctx, m.data, 1, name.c_str())) return rc;
    if (int rc = CheckDeviceBuffer(ctx, m.scales, 1, (name + ": scales").c_str())) return rc;
  }
  return RUYAMD_OK;
}

mxfp4::ConvertCall ConvertOf(const ruyamd_mat& m, const mxfp4::Matrix& matrix) {
  mxfp4::ConvertCall call;
  call.data = m.data;
  call.rs = m.order == RUYAMD_ORDER_COL_MAJOR ? 1 : m.stride;
  call.cs = m.order == RUYAMD_ORDER_ROW_MAJOR ? 1 : m.stride;
  call.type = m.dtype;
  call.rows = m.rows;
  call.matrix = matrix;
  return call;
}

}  // namespace
}  // namespace ruyamd

using namespace ruyamd;

extern "C" int ruyamd_quantize_mxfp4(ruyamd_ctx* ctx, const ruyamd_mat* src, const ruyamd_routing* routing,
                                     const ruyamd_mxfp4_mat* dst) {
  if (!ctx) return RUYAMD_E_INVALID;
  ctx->performance_advisories = 0;
  if (!src || !dst) return Fail(ctx, RUYAMD_E_INVALID, "null argument");
  if (int rc = CheckMatrix(ctx, *src, "src")) return rc;
  mxfp4::Matrix matrix;
  if (int rc = CheckMxFp4(ctx, *dst, "dst", &matrix)) return rc;
  if (routing) {
    if (int rc = CheckRouting(ctx, *routing)) return rc;
    if (src->rows != routing->tokens) return Fail(ctx, RUYAMD_E_INVALID, "shape mismatch: src needs a row to each token");
  } else if (src->rows != dst->rows) {
    return Fail(ctx, RUYAMD_E_INVALID, "shape mismatch: src and dst need the same rows");
  }
  if (src->cols != dst->cols) return Fail(ctx, RUYAMD_E_INVALID, "shape mismatch: src and dst need the same columns");
  mxfp4::ConvertCall call = ConvertOf(*src, matrix);
  if (routing) {
    call.places = routing->places;
    call.top = routing->top;
  }
  const bool nothing = src->rows == 0 || src->cols == 0 || dst->rows == 0 || (routing && routing->top == 0);
  return LaunchChecked(ctx, nothing, [&]() -> hipError_t {
    hipError_t launched = hipSuccess;
    ctx->last_kernel = RUYAMD_KERNEL_TOKENS;
    if (!ctx->force_generic && mxfp4::LaunchQuantize(ctx->stream, call, ctx->multiprocessor_count, &launched)) return launched;
    ctx->last_kernel = RUYAMD_KERNEL_GENERIC;
    return mxfp4::LaunchGenericQuantize(ctx->stream, call);
  });
}

extern "C" int ruyamd_dequantize_mxfp4(ruyamd_ctx* ctx, const ruyamd_mxfp4_mat* src, const ruyamd_mat* dst) {
  if (!ctx) return RUYAMD_E_INVALID;
  ctx->performance_advisories = 0;
  if (!src || !dst) return Fail(ctx, RUYAMD_E_INVALID, "null argument");
  mxfp4::Matrix matrix;
  if (int rc = CheckMxFp4(ctx, *src, "src", &matrix)) return rc;
  if (int rc = CheckMatrix(ctx, *dst, "dst")) return rc;
  if (src->rows != dst->rows || src->cols != dst->cols)
    return Fail(ctx, RUYAMD_E_INVALID, "shape mismatch: src and dst need the same size");
  const mxfp4::ConvertCall call = ConvertOf(*dst, matrix);
  return LaunchChecked(ctx, dst->rows == 0 || dst->cols == 0, [&]() -> hipError_t {
    hipError_t launched = hipSuccess;
    ctx->last_kernel = RUYAMD_KERNEL_TOKENS;
    if (!ctx->force_generic && mxfp4::LaunchDequantize(ctx->stream, call, ctx->multiprocessor_count, &launched)) return launched;
    ctx->last_kernel = RUYAMD_KERNEL_GENERIC;
    return mxfp4::LaunchGenericDequantize(ctx->stream, call);
  });
}

extern "C" int ruyamd_mul_mxfp4(ruyamd_ctx* ctx, const ruyamd_mxfp4_mat* lhs, const ruyamd_mxfp4_mat* rhs,
                                const ruyamd_groups* groups, const ruyamd_mul_params* params, const ruyamd_mat* dst) {
  if (!ctx) return RUYAMD_E_INVALID;
  ctx->performance_advisories = 0;
  if (!lhs || !rhs || !params || !dst) return Fail(ctx, RUYAMD_E_INVALID, "null argument");
  mxfp4::MulCall call;
  if (int rc = CheckMxFp4(ctx, *lhs, "lhs", &call.lhs)) return rc;
  if (int rc = CheckMxFp4(ctx, *rhs, "rhs", &call.rhs)) return rc;
  if (int rc = CheckMatrix(ctx, *dst, "dst")) return rc;
  if (lhs->cols != rhs->cols || dst->rows != lhs->rows || dst->cols != rhs->rows)
    return Fail(ctx, RUYAMD_E_INVALID, "shape mismatch: need lhs MxK, rhs NxK, dst MxN");
  if (groups)
    if (int rc = CheckGroups(ctx, *groups)) return rc;
  if (int rc = CheckParams(ctx, *params, true)) return rc;
  call.dst = dst->data;
  call.dst_rs = dst->order == RUYAMD_ORDER_COL_MAJOR ? 1 : dst->stride;
  call.dst_cs = dst->order == RUYAMD_ORDER_ROW_MAJOR ? 1 : dst->stride;
  call.dst_type = dst->dtype;
  call.m = dst->rows;
  call.n = dst->cols;
  call.k = lhs->cols;
  call.bias = static_cast<const float*>(params->bias);
  call.clamp_min = static_cast<float>(params->clamp_min);
  call.clamp_max = static_cast<float>(params->clamp_max);
  if (groups) {
    call.offsets = groups->offsets;
    call.groups = groups->count;
    call.bias_stride = groups->bias_stride ? groups->bias_stride : dst->rows;
  }
  call.compute_units = ctx->multiprocessor_count;
  call.forced_tile_rows = ctx->forced_tile_rows;
  call.forced_tile_cols = ctx->forced_tile_cols;
  call.forced_deep = ctx->forced_depth_parts != 0;
  return LaunchChecked(ctx, call.m == 0 || call.n == 0, [&]() -> hipError_t {
    hipError_t launched = hipSuccess;
    ctx->last_kernel = RUYAMD_KERNEL_MXFP4_STREAM;
    if (!ctx->force_generic && mxfp4::LaunchStream(ctx->stream, call, &launched)) return launched;
    ctx->last_kernel = RUYAMD_KERNEL_MXFP4_MFMA;
    if (!ctx->force_generic && mxfp4::LaunchTiles(ctx->stream, call, &launched)) return launched;
    ctx->last_kernel = RUYAMD_KERNEL_GENERIC;
    return mxfp4::LaunchGeneric(ctx->stream, call);
  });
}
