// The streaming kernels of weights in the tokens' own type, and the choice of a
// streaming kernel.
#include "grouped_stream.h"
#include <cstdlib>

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

  // Tokens of all depth in LDS where 16 of them (or as many as there are) fit, and
  // slab by slab otherwise; tokens whose values do not lie side by side as many as fit.
  const int depth_to_chunk = int4 ? 256 : 128 / bytes;
  const int64_t whole_pitch = int64_t((call.k + depth_to_chunk - 1) / depth_to_chunk) * (int4 ? 512 : 128) + 16;
  const int64_t room = 128 << 10;
  const int64_t fit = room / (whole_pitch * rows_to_token);
  const int64_t to_group = call.offsets ? block_tokens : call.n;  // (a group may have many more than others)
  if (call.rhs_rs != 1) {
    if (fit == 0) return false;
    plan.cols = 1;
    plan.slabs = false;
  } else {
    plan.cols = per_group <= block_tokens ? 1 : per_group <= 2 * block_tokens || !int4 ? 2 : 4;
    plan.slabs = plan.cols > 1 || min(to_group, int64_t(block_tokens)) > fit;
  }
  const int chunk = int4 && plan.slabs ? 128 : depth_to_chunk, chunks = (call.k + chunk - 1) / chunk;
  const int chunk_bytes = int4 ? 2 * chunk : 128;  // of a token in LDS
  args.tokens = static_cast<int>(plan.slabs ? plan.cols * block_tokens : min(fit, int64_t(block_tokens)));

  plan.scaling = Scaling::kWide;
  args.scale_shift = 31;
  if (int4 && weights->group_size < call.k) {
    const int size = weights->group_size, scales = (call.k + size - 1) / size;
    args.scale_shift = __builtin_ctz(size);
    plan.scaling = size >= 128 && (size & (size - 1)) == 0 ? Scaling::kWide
                   : size == 64 && scales >= chunk / 64    ? Scaling::k64
                   : size == 32 && scales >= chunk / 32    ? Scaling::k32
                                                           : Scaling::kAny;
  }

  // Waves: 16 to a CU if the rows give them, 8 to a workgroup, along the rows first, then
  // along the depth.
  int row_waves = RowWaves(plan.slabs, plan.cols), depth_waves = 8 / row_waves;
  plan.rows = plan.slabs || plan.scaling == Scaling::kAny ? 1 : 2;
  if (const char* e = getenv("S_ROWS")) if (plan.rows == 2) plan.rows = atoi(e);
  while (plan.rows > 1 && (call.m + 16 * plan.rows * row_waves - 1) / (16 * plan.rows * row_waves) * busy < call.compute_units)
    plan.rows /= 2;
  if (!plan.slabs) {
    const int64_t units = (call.m + 16 * plan.rows - 1) / (16 * plan.rows) * busy;
    int per_cu = 16;
    if (const char* e = getenv("S_WAVES")) per_cu = atoi(e);
    while (depth_waves > 1 && units * depth_waves > int64_t(per_cu) * call.compute_units) depth_waves /= 2;
    row_waves = 8 / depth_waves;
  }
  while (depth_waves > 1 && chunks < depth_waves) depth_waves /= 2;
  plan.waves = depth_waves * row_waves;
  args.depth_waves = depth_waves;
  args.row_waves = row_waves;
  const int work_rows = 16 * plan.rows * row_waves;
  args.tiles_m = (call.m + work_rows - 1) / work_rows;
  const int64_t slots = call.offsets ? call.n / args.tokens + busy : (call.n + args.tokens - 1) / args.tokens;
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
    lds = min(int64_t(args.tokens), to_group) * rows_to_token * whole_pitch;
  }
  const int64_t sums = int64_t(plan.waves) * plan.rows * 1024;
  plan.lds_bytes = static_cast<unsigned>(lds > sums ? lds : sums);

  if (int4) {
    *status = call.type == RUYAMD_DTYPE_BF16  ? LaunchStreamInt4Bf16(stream, args, plan)
              : call.type == RUYAMD_DTYPE_F16 ? LaunchStreamInt4F16(stream, args, plan)
                                              : LaunchStreamInt4F32(stream, args, plan);
  } else {
    *status = call.type == RUYAMD_DTYPE_BF16  ? LaunchStreamFloat<RUYAMD_DTYPE_BF16>(stream, args, plan)
              : call.type == RUYAMD_DTYPE_F16 ? LaunchStreamFloat<RUYAMD_DTYPE_F16>(stream, args, plan)
                                              : LaunchStreamFloat<RUYAMD_DTYPE_F32>(stream, args, plan);
  }
  return true;
}

}  // namespace grouped
}  // namespace ruyamd
