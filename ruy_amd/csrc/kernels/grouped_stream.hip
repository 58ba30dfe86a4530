// The streaming kernels of weights in the tokens' own type, and the choice of a
// streaming kernel.
#include "grouped_stream.h"
#include "launch_geometry.h"

namespace ruyamd {
namespace grouped {

bool LaunchStream(hipStream_t stream, const Call& call, const Int4* weights, hipError_t* status) {
  const bool int4 = weights != nullptr;
  if (!int4 && (call.dealt != Dealt::kColumns || call.lhs_cs != 1 || call.forced_tile_rows)) return false;
  // (A row has 16 bytes at least, and what a lane has of one ends before 2^31.)
  if (call.k < 32 || call.k > (1 << 28)) return false;
  // (Sizes are rounded up to workgroups in 32 bits.)
  if (max(call.m, call.n) > 0x7fffffff - 2048) return false;
  StreamArgs args;
  args.c = call;
  if (int4) args.w = *weights;
  const bool parts = int4 && call.type == RUYAMD_DTYPE_F32;
  const int bytes = call.type == RUYAMD_DTYPE_F32 ? 4 : 2;
  const int block_tokens = parts ? 5 : 16, rows_to_token = parts ? 3 : 1;
  const int64_t busy = min(call.groups, call.n);
  const int64_t per_group = (call.n + busy - 1) / busy;
  // (Weights in the tokens' type: up to 32 columns a group, in the mean over groups. Streaming and tiles, us, weights out of
  // HBM: bfloat16 1 x 4096x4096, 16 columns 11.2 and 20.0, 32 17.4 and 20.7; 64 x 2048x2048, 1 a group 90 and 98, 8 102 and 101, 32
  // 129 and 104; fp32 8 x 1024x1024, 16 16.3 and 21.1, 32 14.4 and 21.1; 64 x 512x1024, 16 54.7 and 37.9, 32 38.4 and 38.9.
  // The line is right for few groups, about right for fp32, and late for 16 bits where the groups' weights make some hundred tiles: 8 x
  // 4096x2048 1 31.3 and 31.2, 16 51.0 and 30.8, 32 35.5 and 30.9; 16 x 1024x1024 1 12.7 and 9.1, 32 13.0 and 9.6.)
  if (!int4 && per_group > 32) return false;
  StreamPlan plan;

  // Tokens of all depth in LDS where 16 of them (or as many as there are) fit, and
  // slab by slab otherwise; tokens whose values do not lie side by side as many as fit.
  const int depth_to_chunk = int4 ? 256 : 128 / bytes;
  const int64_t whole_pitch = int64_t((call.k + depth_to_chunk - 1) / depth_to_chunk) * (int4 ? 512 : 128) + 16;
  const int64_t room = 128 << 10;
  const int64_t fit = room / (whole_pitch * rows_to_token);
  // (A group may have more than its share: room for four times as many, which several
  // workgroups then read the weights for where it has more still.)
  const int64_t to_group = call.offsets ? min(int64_t(block_tokens), 4 * per_group) : call.n;
  if (call.rhs_rs != 1) {
    if (fit == 0) return false;
    plan.cols = 1;
    plan.slabs = false;
  } else {
    plan.cols = per_group <= block_tokens ? 1 : 2;
    plan.slabs = plan.cols > 1 || min(to_group, int64_t(block_tokens)) > fit;
  }
  const int chunk = int4 && plan.slabs ? 128 : depth_to_chunk, chunks = (call.k + chunk - 1) / chunk;
  const int chunk_bytes = int4 ? 2 * chunk : 128;  // of a token in LDS
  args.tokens = static_cast<int>(plan.slabs ? plan.cols * block_tokens : min(fit, min(int64_t(block_tokens), to_group)));

  plan.scaling = Scaling::kWide;
  args.scale_shift = 31;
  if (int4 && weights->group_size < call.k) {
    const int size = weights->group_size;
    args.scale_shift = __builtin_ctz(size);
    plan.scaling = size >= 128 && (size & (size - 1)) == 0 ? Scaling::kWide
                   : size == 64                            ? Scaling::k64
                   : size == 32                            ? Scaling::k32
                                                           : Scaling::kAny;
  }

  // Waves: 8 to a workgroup, along the depth as long as that makes no more than 16 to a CU
  // (of weights in 16 or 32 bits 64), along the rows otherwise; fewer rows where what goes with
  // them into LDS is too much. (Half, 64 x 2048x2048, 32 tokens: 64 waves to a CU
  // 40.6 us, 16 44.0. 4-bit, the same: 24.9 and 22.5; 16384 x 16384, one token: 31.5 and
  // 30.7, with 4 waves to a workgroup 40, with 2 59. Two blocks of 16 rows to a wave are no
  // faster anywhere, and slower where there are few rows.)
  int row_waves = RowWaves(plan.slabs, plan.cols), depth_waves = 8 / row_waves;
  if (!plan.slabs) {
    const int64_t units = (int64_t(call.m) + 15) / 16 * busy;
    const int64_t most = int64_t(int4 ? 16 : 64) * call.compute_units;
    depth_waves = 8;
    while (depth_waves > 1 && units * depth_waves > most) depth_waves /= 2;
    row_waves = 8 / depth_waves;
  }
  while (depth_waves > 1 && chunks < depth_waves) depth_waves /= 2;
  const int padded_scales = chunks * (chunk / (plan.scaling == Scaling::kWide ? 128 : plan.scaling == Scaling::k64 ? 64 : 32));
  // (Odd numbers of words: 16 rows side by side reach 16 banks.)
  args.scale_pitch = padded_scales | 1;
  args.zero_pitch = ((padded_scales + 3) / 4 | 1) * 4;
  int64_t tokens_lds = 0, scales_lds = 0, zeros_lds = 0;
  const int64_t lost_lds = parts ? 8 * sizeof(int) : 0;  // (for 8 waves, the most there are)
  int work_rows = 0;
  for (;;) {
    work_rows = 16 * row_waves;
    if (plan.slabs) {
      args.pitch = depth_waves * chunk_bytes + 16;
      args.slab_bytes = 16 * plan.cols * args.pitch;
      tokens_lds = 2 * args.slab_bytes;
    } else {
      args.pitch = static_cast<int>(whole_pitch);
      args.slab_bytes = 0;
      tokens_lds = int64_t(args.tokens) * rows_to_token * whole_pitch;
    }
    if (int4 && plan.scaling != Scaling::kAny) {
      scales_lds = int64_t(work_rows) * args.scale_pitch * 4;
      zeros_lds = weights->zero_points ? int64_t(work_rows) * args.zero_pitch : 0;
    }
    if (tokens_lds + scales_lds + zeros_lds + lost_lds <= kStreamLds) break;
    if (!plan.slabs && row_waves > 1) {
      row_waves /= 2;
      if (depth_waves * 2 <= chunks) depth_waves *= 2;
    } else if (plan.slabs && depth_waves > 1) {
      depth_waves /= 2;
    } else {
      plan.scaling = Scaling::kAny;
      scales_lds = zeros_lds = 0;
    }
  }
  args.scales_at = static_cast<int>(tokens_lds);
  args.zeros_at = static_cast<int>(tokens_lds + scales_lds);
  args.lost_at = static_cast<int>(tokens_lds + scales_lds + zeros_lds);
  plan.waves = depth_waves * row_waves;
  args.depth_waves = depth_waves;
  args.row_waves = row_waves;
  args.tiles_m = (call.m + work_rows - 1) / work_rows;
  const int64_t lds = tokens_lds + scales_lds + zeros_lds + lost_lds, sums = int64_t(plan.waves) * 1024;
  plan.lds_bytes = static_cast<unsigned>(lds > sums ? lds : sums);
  const int64_t slots = call.offsets ? call.n / args.tokens + busy : (call.n + args.tokens - 1) / args.tokens;
  const int64_t blocks = (slots * args.tiles_m + 7) / 8 * 8;
  if (!LaunchFits(blocks, 64 * plan.waves)) return false;
  plan.blocks = static_cast<unsigned>(blocks);

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
