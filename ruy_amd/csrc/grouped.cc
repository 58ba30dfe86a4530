// ruyamd_mul_grouped, ruyamd_mul_grouped_depth and ruyamd_mul_int4: the checks
// of a call, the choice of its kernel, and its launch on the context's stream.
#include <string>

#include "checks.h"
#include "context.h"
#include "internal.h"
#include "kernels/grouped.h"

namespace ruyamd {
namespace {

using grouped::Dealt;

int64_t Extent(const ruyamd_mat& m) {
  const int64_t outer = m.order == RUYAMD_ORDER_COL_MAJOR ? m.cols : m.rows;
  return outer * m.stride;
}

// Both sides, dst and what they have to agree in. `lhs_rows` x `depth` is the left-hand operand.
int CheckTypesAndShape(ruyamd_ctx* ctx, int lhs_type, int lhs_rows, int lhs_cols, const ruyamd_mat& rhs,
                       const ruyamd_mat& dst) {
  if (lhs_cols != rhs.rows || dst.rows != lhs_rows || dst.cols != rhs.cols)
    return Fail(ctx, RUYAMD_E_INVALID, "shape mismatch: need lhs MxK, rhs KxN, dst MxN");
  if (lhs_type != rhs.dtype) return Fail(ctx, RUYAMD_E_UNSUPPORTED, "both operands must have the same type");
  if (dst.dtype != rhs.dtype && dst.dtype != RUYAMD_DTYPE_F32)
    return Fail(ctx, RUYAMD_E_UNSUPPORTED, "dst must have the operands' type or be fp32");
  return RUYAMD_OK;
}

void SetMatrices(const ruyamd_mat& rhs, const ruyamd_mat& dst, const ruyamd_mul_params& p, const ruyamd_groups* groups,
                 grouped::Call* call) {
  const auto strides = [](const ruyamd_mat& m, int64_t* rs, int64_t* cs) {
    *rs = m.order == RUYAMD_ORDER_COL_MAJOR ? 1 : m.stride;
    *cs = m.order == RUYAMD_ORDER_ROW_MAJOR ? 1 : m.stride;
  };
  call->rhs = rhs.data;
  call->dst = dst.data;
  strides(rhs, &call->rhs_rs, &call->rhs_cs);
  strides(dst, &call->dst_rs, &call->dst_cs);
  call->m = dst.rows;
  call->n = dst.cols;
  call->k = rhs.rows;
  call->type = rhs.dtype;
  call->dst_type = dst.dtype;
  call->bias = static_cast<const float*>(p.bias);
  call->clamp_min = static_cast<float>(p.clamp_min);
  call->clamp_max = static_cast<float>(p.clamp_max);
  if (!groups) return;
  call->offsets = groups->offsets;
  call->groups = groups->count;
  call->bias_stride = groups->bias_stride ? groups->bias_stride : dst.rows;
}

// Launches a checked call.
int Run(ruyamd_ctx* ctx, grouped::Call* call, const grouped::Int4* weights) {
  call->compute_units = ctx->multiprocessor_count;
  call->forced_tile_rows = ctx->forced_tile_rows;
  call->forced_tile_cols = ctx->forced_tile_cols;
  return LaunchChecked(ctx, call->m == 0 || call->n == 0, [&]() -> hipError_t {
    hipError_t launched = hipSuccess;
    if (!ctx->force_generic && grouped::LaunchStream(ctx->stream, *call, weights, &launched)) {
      ctx->last_kernel = weights ? RUYAMD_KERNEL_INT4_STREAM : RUYAMD_KERNEL_GROUPED_STREAM;
    } else if (!ctx->force_generic && !weights && grouped::LaunchTiles(ctx->stream, *call, &launched)) {
      ctx->last_kernel = RUYAMD_KERNEL_GROUPED_MFMA;
    } else {
      launched = grouped::LaunchGeneric(ctx->stream, *call, weights);
      ctx->last_kernel = RUYAMD_KERNEL_GENERIC;
    }
    return launched;
  });
}

int MulGrouped(ruyamd_ctx* ctx, Dealt dealt, const ruyamd_mat* lhs, const ruyamd_mat* rhs, const ruyamd_groups* groups,
               const ruyamd_mul_params* p, const ruyamd_mat* dst) {
  if (!ctx) return RUYAMD_E_INVALID;
  ctx->performance_advisories = 0;
  if (!lhs || !rhs || !groups || !p || !dst) return Fail(ctx, RUYAMD_E_INVALID, "null argument");
  if (int rc = CheckMatrix(ctx, *lhs, "lhs")) return rc;
  if (int rc = CheckMatrix(ctx, *rhs, "rhs")) return rc;
  if (int rc = CheckMatrix(ctx, *dst, "dst")) return rc;
  if (int rc = CheckTypesAndShape(ctx, lhs->dtype, lhs->rows, lhs->cols, *rhs, *dst)) return rc;
  if (int rc = CheckGroups(ctx, *groups)) return rc;
  if (int rc = CheckParams(ctx, *p, dealt == Dealt::kColumns)) return rc;
  grouped::Call call;
  call.dealt = dealt;
  SetMatrices(*rhs, *dst, *p, groups, &call);
  call.lhs = lhs->data;
  call.lhs_rs = lhs->order == RUYAMD_ORDER_COL_MAJOR ? 1 : lhs->stride;
  call.lhs_cs = lhs->order == RUYAMD_ORDER_ROW_MAJOR ? 1 : lhs->stride;
  call.matrix_stride = groups->matrix_stride ? groups->matrix_stride : Extent(dealt == Dealt::kColumns ? *lhs : *dst);
  return Run(ctx, &call, nullptr);
}

}  // namespace
}  // namespace ruyamd

using namespace ruyamd;

extern "C" int ruyamd_mul_grouped(ruyamd_ctx* ctx, const ruyamd_mat* lhs, const ruyamd_mat* rhs,
                                  const ruyamd_groups* groups, const ruyamd_mul_params* params,
                                  const ruyamd_mat* dst) {
  return MulGrouped(ctx, Dealt::kColumns, lhs, rhs, groups, params, dst);
}

extern "C" int ruyamd_mul_grouped_depth(ruyamd_ctx* ctx, const ruyamd_mat* lhs, const ruyamd_mat* rhs,
                                        const ruyamd_groups* groups, const ruyamd_mul_params* params,
                                        const ruyamd_mat* dst) {
  return MulGrouped(ctx, Dealt::kDepth, lhs, rhs, groups, params, dst);
}

extern "C" int ruyamd_mul_int4(ruyamd_ctx* ctx, const ruyamd_int4_mat* lhs, const ruyamd_mat* rhs,
                               const ruyamd_groups* groups, const ruyamd_mul_params* params, const ruyamd_mat* dst) {
  if (!ctx) return RUYAMD_E_INVALID;
  ctx->performance_advisories = 0;
  if (!lhs || !rhs || !params || !dst) return Fail(ctx, RUYAMD_E_INVALID, "null argument");
  if (lhs->rows < 0 || lhs->cols < 0) return Fail(ctx, RUYAMD_E_INVALID, "lhs: negative size");
  if (int rc = CheckMatrix(ctx, *rhs, "rhs")) return rc;
  if (int rc = CheckMatrix(ctx, *dst, "dst")) return rc;
  if (int rc = CheckTypesAndShape(ctx, rhs->dtype, lhs->rows, lhs->cols, *rhs, *dst)) return rc;
  if (groups)
    if (int rc = CheckGroups(ctx, *groups)) return rc;
  if (int rc = CheckParams(ctx, *params, true)) return rc;
  grouped::Int4 w;
  if (lhs->group_size < 1 || (lhs->group_size % 32 && lhs->group_size < lhs->cols))
    return Fail(ctx, RUYAMD_E_INVALID, "lhs: group_size must be a multiple of 32, or at least cols");
  if (!IsOperandType(lhs->scale_dtype))
    return Fail(ctx, RUYAMD_E_UNSUPPORTED, "lhs: scales must be fp32, bfloat16 or half");
  if (lhs->row_bytes < 0 || lhs->scale_stride < 0 || lhs->matrix_bytes < 0 || lhs->scales_matrix_stride < 0)
    return Fail(ctx, RUYAMD_E_INVALID, "lhs: negative stride");
  const int64_t bytes = (int64_t(lhs->cols) + 1) / 2;
  const int64_t scales = (int64_t(lhs->cols) + lhs->group_size - 1) / lhs->group_size;
  w.row_bytes = lhs->row_bytes ? lhs->row_bytes : bytes;
  w.scale_stride = lhs->scale_stride ? lhs->scale_stride : scales;
  if (w.row_bytes < bytes || w.scale_stride < scales)
    return Fail(ctx, RUYAMD_E_INVALID, "lhs: stride smaller than a row");
  w.matrix_bytes = lhs->matrix_bytes ? lhs->matrix_bytes : w.row_bytes * lhs->rows;
  w.scales_matrix_stride = lhs->scales_matrix_stride ? lhs->scales_matrix_stride : w.scale_stride * lhs->rows;
  if (lhs->rows > 0 && lhs->cols > 0) {
    if (int rc = CheckDeviceBuffer(ctx, lhs->data, 1, "lhs")) return rc;
    if (int rc = CheckDeviceBuffer(ctx, lhs->scales, lhs->scale_dtype == RUYAMD_DTYPE_F32 ? 4 : 2, "lhs: scales")) return rc;
    if (lhs->zero_points)
      if (int rc = CheckDeviceBuffer(ctx, lhs->zero_points, 1, "lhs: zero points")) return rc;
  }
  w.data = static_cast<const uint8_t*>(lhs->data);
  w.scales = lhs->scales;
  w.zero_points = lhs->zero_points;
  w.group_size = lhs->group_size;
  w.scale_type = lhs->scale_dtype;
  grouped::Call call;
  SetMatrices(*rhs, *dst, *params, groups, &call);
  return Run(ctx, &call, &w);
}
