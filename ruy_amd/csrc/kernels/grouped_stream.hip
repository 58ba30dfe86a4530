// The streaming kernels of weights in the tokens' own type, and the choice of a
// streaming kernel.
#include "grouped_stream.h"

namespace ruyamd {
namespace grouped {

bool LaunchStream(hipStream_t stream, const Call& call, const Int4* weights, hipError_t* status) {
  const bool int4 = weights != nullptr;
  if (!int4 && (call.dealt != Dealt::kColumns || call.lhs_cs != 1)) return false;
  // (A row has 16 bytes at least, and what a lane has of one ends before 2^31.)
  if (call.k < 32 || call.k > (1 << 28)) return false;
  StreamArgs args;
  args.c = call;
  if (int4) args.w = *weights;
  const bool parts = int4 && call.type == RUYAMD_DTYPE_F32;
  const int bytes = call.type == RUYAMD_DTYPE_F32 ? 4 : 2;
  const int block_tokens = parts ? 5 : 16, rows_to_token = parts ? 3 : 1;
  const int64_t busy = min(call.groups, call.n);
  const int64_t per_group = (call.n + busy - 1) / busy;
  if (!int4 && per_group > 32) return false;
  StreamPlan plan;
  plan.cols = per_group <= block_tokens ? 1 : per_group <= 2 * block_tokens ? 2 : 4;
  if (!int4) plan.cols = min(plan.cols, 2);

  const int chunk = int4 ? 128 : 128 / bytes;              // depth positions
  const int chunk_bytes = int4 ? 256 : 128;                // of a token in LDS
  const int chunks = (call.k + chunk - 1) / chunk;
  plan.scaling = Scaling::kWide;
  if (int4 && weights->group_size < call.k && weights->group_size % 128) {
    const int scales = (call.k + weights->group_size - 1) / weights->group_size;
    plan.scaling = weights->group_size == 64 && scales >= 2   ? Scaling::k64
                   : weights->group_size == 32 && scales >= 4 ? Scaling::k32
                                                              : Scaling::kAny;
  }

  // Tokens of all depth in LDS where they fit.
  const int64_t most = min(int64_t(block_tokens), call.offsets ? int64_t(block_tokens) : int64_t(call.n)) * rows_to_token;
  const int64_t whole_pitch = int64_t(chunks) * chunk_bytes + 16;
  plan.slabs = plan.cols > 1 || most * whole_pitch > (128 << 10);

  const int row_waves = RowWaves(plan.slabs, plan.cols);
  plan.rows = plan.cols > 2 ? 1 : plan.cols > 1 || int4 ? 2 : 4;
  if (plan.scaling == Scaling::kAny) plan.rows = 1;
  while (plan.rows > 1 && (call.m + 16 * plan.rows * row_waves - 1) / (16 * plan.rows * row_waves) * busy < call.compute_units)
    plan.rows /= 2;
  int depth_waves = 8 / row_waves;
  while (depth_waves > 1 && chunks < depth_waves) depth_waves /= 2;
  plan.waves = depth_waves * row_waves;
  args.depth_waves = depth_waves;
  const int work_rows = 16 * plan.rows * row_waves;
  args.tiles_m = (call.m + work_rows - 1) / work_rows;
  const int64_t work_tokens = plan.cols * block_tokens;
  const int64_t slots = call.offsets ? call.n / work_tokens + busy : (call.n + work_tokens - 1) / work_tokens;
  const int64_t blocks = (slots * args.tiles_m + 7) / 8 * 8;
  if (blocks > 0x7fffffff) return false;
  plan.blocks = static_cast<unsigned>(blocks);

  int64_t lds;
  if (plan.slabs) {
    args.pitch = depth_waves * chunk_bytes + 16;
    args.slab_bytes = 16 * plan.cols * args.pitch;
    lds = 2 * args.slab_bytes;
  } else {
    args.pitch = static_cast<int>(whole_pitch);
    args.slab_bytes = 0;
    lds = most * whole_pitch;
  }
  const int64_t sums = int64_t(plan.waves) * plan.rows * 1024;
  plan.lds_bytes = static_cast<unsigned>(lds > sums ? lds : sums);

  if (int4) {
    *status = call.type == RUYAMD_DTYPE_BF16  ? LaunchStreamInt4Bf16(stream, args, plan)
              : call.type == RUYAMD_DTYPE_F16 ? LaunchStreamInt4F16(stream, args, plan)
                                              : LaunchStreamInt4F32(stream, args, plan);
  } else {
    *status = call.type == RUYAMD_DTYPE_BF16  ? LaunchStreamScaling<false, RUYAMD_DTYPE_BF16, Scaling::kWide>(stream, args, plan)
              : call.type == RUYAMD_DTYPE_F16 ? LaunchStreamScaling<false, RUYAMD_DTYPE_F16, Scaling::kWide>(stream, args, plan)
                                              : LaunchStreamScaling<false, RUYAMD_DTYPE_F32, Scaling::kWide>(stream, args, plan);
  }
  return true;
}

}  // namespace grouped
}  // namespace ruyamd
