// ruyamd_sort_tokens, ruyamd_dispatch_tokens, ruyamd_combine_tokens and
// ruyamd_combine_tokens_gradients: the checks of a call and its launch on the
// context's stream.
#include "kernels/routing.h"

#include <string>

#include "checks.h"
#include "context.h"
#include "internal.h"

namespace ruyamd {

int CheckRouting(ruyamd_ctx* ctx, const ruyamd_routing& r) {
  if (r.tokens < 0 || r.top < 0) return Fail(ctx, RUYAMD_E_INVALID, "routing: negative size");
  if (int64_t(r.tokens) * r.top > 0x7fffffff) return Fail(ctx, RUYAMD_E_UNSUPPORTED, "routing: 2^31 choices or more");
  if (r.count < 1 || r.count > kMostGroups) return Fail(ctx, RUYAMD_E_INVALID, "routing: count must be 1 .. 65536");
  if (r.tokens > 0 && r.top > 0) return CheckDeviceBuffer(ctx, r.places, 4, "routing: places");
  return RUYAMD_OK;
}

namespace {

routing::View ViewOf(const ruyamd_mat& m) {
  return {m.data, m.order == RUYAMD_ORDER_COL_MAJOR ? 1 : m.stride, m.order == RUYAMD_ORDER_ROW_MAJOR ? 1 : m.stride, m.dtype};
}

int CheckWeights(ruyamd_ctx* ctx, const ruyamd_mat& m, const ruyamd_routing& r, const char* name) {
  if (int rc = CheckMatrix(ctx, m, name)) return rc;
  if (m.rows != r.top || m.cols != r.tokens)
    return Fail(ctx, RUYAMD_E_INVALID, std::string(name) + ": must be top x tokens");
  return RUYAMD_OK;
}

// The checked matrices of a call: a column to each token and a column to each place.
int SetSides(ruyamd_ctx* ctx, const ruyamd_routing& r, const ruyamd_mat& token_side, const ruyamd_mat& place_side,
             routing::Call* call) {
  if (token_side.cols != r.tokens) return Fail(ctx, RUYAMD_E_INVALID, "shape mismatch: need a column to each token");
  if (token_side.rows != place_side.rows) return Fail(ctx, RUYAMD_E_INVALID, "shape mismatch: need columns of one length");
  call->places = r.places;
  call->tokens = r.tokens;
  call->top = r.top;
  call->width = token_side.rows;
  call->columns = place_side.cols;
  call->token_side = ViewOf(token_side);
  call->place_side = ViewOf(place_side);
  return RUYAMD_OK;
}

// fast and generic: launches of either kind of kernels.
template <class Fast, class Generic>
int Run(ruyamd_ctx* ctx, bool nothing, Fast&& fast, Generic&& generic) {
  return LaunchChecked(ctx, nothing, [&]() -> hipError_t {
    hipError_t launched = hipSuccess;
    ctx->last_kernel = RUYAMD_KERNEL_TOKENS;
    if (!ctx->force_generic && fast(&launched)) return launched;
    ctx->last_kernel = RUYAMD_KERNEL_GENERIC;
    return generic();
  });
}

}  // namespace
}  // namespace ruyamd

using namespace ruyamd;

extern "C" int ruyamd_sort_tokens(ruyamd_ctx* ctx, const ruyamd_mat* experts, const ruyamd_routing* routing) {
  if (!ctx) return RUYAMD_E_INVALID;
  ctx->performance_advisories = 0;
  if (!experts || !routing) return Fail(ctx, RUYAMD_E_INVALID, "null argument");
  const ruyamd_mat& e = *experts;
  if (int rc = CheckRouting(ctx, *routing)) return rc;
  if (e.order != RUYAMD_ORDER_COL_MAJOR && e.order != RUYAMD_ORDER_ROW_MAJOR)
    return Fail(ctx, RUYAMD_E_INVALID, "experts: bad order");
  if (e.dtype != RUYAMD_DTYPE_I32 && e.dtype != RUYAMD_DTYPE_I64)
    return Fail(ctx, RUYAMD_E_UNSUPPORTED, "experts: the type must be int32 or int64");
  if (e.zero_point) return Fail(ctx, RUYAMD_E_INVALID, "experts: zero_point must be 0");
  if (e.rows != routing->top || e.cols != routing->tokens)
    return Fail(ctx, RUYAMD_E_INVALID, "experts: must be top x tokens");
  if (e.stride < (e.order == RUYAMD_ORDER_COL_MAJOR ? e.rows : e.cols))
    return Fail(ctx, RUYAMD_E_INVALID, "experts: stride smaller than the contiguous dimension");
  if (int rc = CheckDeviceBuffer(ctx, routing->offsets, 4, "routing: offsets")) return rc;
  if (e.rows > 0 && e.cols > 0) {
    if (int rc = CheckDeviceBuffer(ctx, e.data, e.dtype == RUYAMD_DTYPE_I64 ? 8 : 4, "experts")) return rc;
    if (routing->sources)
      if (int rc = CheckDeviceBuffer(ctx, routing->sources, 4, "routing: sources")) return rc;
  }
  routing::SortCall call;
  call.experts = e.data;
  call.rs = e.order == RUYAMD_ORDER_COL_MAJOR ? 1 : e.stride;
  call.cs = e.order == RUYAMD_ORDER_ROW_MAJOR ? 1 : e.stride;
  call.wide = e.dtype == RUYAMD_DTYPE_I64;
  call.tokens = routing->tokens;
  call.top = routing->top;
  call.count = routing->count;
  call.offsets = routing->offsets;
  call.places = routing->places;
  call.sources = routing->sources;
  return LaunchChecked(ctx, false, [&]() -> hipError_t {
    ctx->last_kernel = RUYAMD_KERNEL_TOKENS;
    return routing::LaunchSort(ctx->stream, call, ctx->force_generic);
  });
}

extern "C" int ruyamd_dispatch_tokens(ruyamd_ctx* ctx, const ruyamd_mat* src, const ruyamd_routing* routing,
                                      const ruyamd_mat* dst) {
  if (!ctx) return RUYAMD_E_INVALID;
  ctx->performance_advisories = 0;
  if (!src || !routing || !dst) return Fail(ctx, RUYAMD_E_INVALID, "null argument");
  if (int rc = CheckRouting(ctx, *routing)) return rc;
  if (int rc = CheckMatrix(ctx, *src, "src")) return rc;
  if (int rc = CheckMatrix(ctx, *dst, "dst")) return rc;
  if (src->dtype != dst->dtype) return Fail(ctx, RUYAMD_E_UNSUPPORTED, "dst must have src's type");
  routing::Call call;
  if (int rc = SetSides(ctx, *routing, *src, *dst, &call)) return rc;
  const bool nothing = call.tokens == 0 || call.top == 0 || call.width == 0 || call.columns == 0;
  return Run(
      ctx, nothing, [&](hipError_t* status) { return routing::LaunchDispatch(ctx->stream, call, ctx->multiprocessor_count, status); },
      [&] { return routing::LaunchGenericDispatch(ctx->stream, call); });
}

extern "C" int ruyamd_combine_tokens(ruyamd_ctx* ctx, const ruyamd_mat* src, const ruyamd_routing* routing,
                                     const ruyamd_mat* weights, const ruyamd_mat* dst) {
  if (!ctx) return RUYAMD_E_INVALID;
  ctx->performance_advisories = 0;
  if (!src || !routing || !dst) return Fail(ctx, RUYAMD_E_INVALID, "null argument");
  if (int rc = CheckRouting(ctx, *routing)) return rc;
  if (int rc = CheckMatrix(ctx, *src, "src")) return rc;
  if (int rc = CheckMatrix(ctx, *dst, "dst")) return rc;
  if (dst->dtype != src->dtype && dst->dtype != RUYAMD_DTYPE_F32)
    return Fail(ctx, RUYAMD_E_UNSUPPORTED, "dst must have src's type or be fp32");
  routing::Call call;
  if (int rc = SetSides(ctx, *routing, *dst, *src, &call)) return rc;
  if (weights) {
    if (int rc = CheckWeights(ctx, *weights, *routing, "weights")) return rc;
    call.weights = ViewOf(*weights);
  }
  return Run(
      ctx, call.tokens == 0 || call.width == 0,
      [&](hipError_t* status) { return routing::LaunchCombine(ctx->stream, call, ctx->multiprocessor_count, status); },
      [&] { return routing::LaunchGenericCombine(ctx->stream, call); });
}

extern "C" int ruyamd_combine_tokens_gradients(ruyamd_ctx* ctx, const ruyamd_mat* grad, const ruyamd_mat* src,
                                               const ruyamd_routing* routing, const ruyamd_mat* weights,
                                               const ruyamd_mat* grad_src, const ruyamd_mat* grad_weights) {
  if (!ctx) return RUYAMD_E_INVALID;
  ctx->performance_advisories = 0;
  if (!grad || !routing) return Fail(ctx, RUYAMD_E_INVALID, "null argument");
  if (!grad_src && !grad_weights) return Fail(ctx, RUYAMD_E_INVALID, "no gradient is asked for");
  if (grad_weights && !src) return Fail(ctx, RUYAMD_E_INVALID, "grad_weights needs src");
  if (int rc = CheckRouting(ctx, *routing)) return rc;
  if (int rc = CheckMatrix(ctx, *grad, "grad")) return rc;
  if (src)
    if (int rc = CheckMatrix(ctx, *src, "src")) return rc;
  if (grad_src) {
    if (int rc = CheckMatrix(ctx, *grad_src, "grad_src")) return rc;
    if (src && (grad_src->dtype != src->dtype || grad_src->rows != src->rows || grad_src->cols != src->cols))
      return Fail(ctx, RUYAMD_E_INVALID, "grad_src must have src's type and size");
  }
  const ruyamd_mat& rows = src ? *src : *grad_src;
  if (grad->dtype != rows.dtype && grad->dtype != RUYAMD_DTYPE_F32)
    return Fail(ctx, RUYAMD_E_UNSUPPORTED, "grad must have src's type or be fp32");
  routing::Call call;
  if (int rc = SetSides(ctx, *routing, *grad, rows, &call)) return rc;
  if (weights && grad_src) {
    if (int rc = CheckWeights(ctx, *weights, *routing, "weights")) return rc;
    call.weights = ViewOf(*weights);
  }
  // (A gradient that has no elements is none that is wanted.)
  if (grad_src && call.width && call.columns) call.grad_src = ViewOf(*grad_src);
  if (grad_weights) {
    if (int rc = CheckWeights(ctx, *grad_weights, *routing, "grad_weights")) return rc;
    call.grad_weights = ViewOf(*grad_weights);
  }
  return Run(
      ctx, call.tokens == 0 || call.top == 0 || (!call.grad_src.data && !call.grad_weights.data),
      [&](hipError_t* status) { return routing::LaunchGradients(ctx->stream, call, ctx->multiprocessor_count, status); },
      [&] { return routing::LaunchGenericGradients(ctx->stream, call); });
}
