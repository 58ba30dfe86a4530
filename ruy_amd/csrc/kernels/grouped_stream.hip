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
  const int block_tokens = parts ? 5 : 16;
  const int64_t busy = min(call.groups, call.n);
  const int64_t per_group = (call.n + busy - 1) / busy;
  if (!int4 && per_group > 32) return false;
  const int cols = per_group <= block_tokens ? 1 : per_group <= 2 * block_tokens ? 2 : 4;
  const int64_t slots = call.n / (cols * block_tokens) + busy;
  int rows = 4 / cols;
  while (rows > 1 && ((call.m + 16 * rows - 1) / (16 * rows)) * busy < call.compute_units) rows /= 2;
  args.row_blocks = (call.m + 16 * rows - 1) / (16 * rows);
  const int64_t blocks = (slots * args.row_blocks + 7) / 8 * 8;
  if (blocks > 0x7fffffff) return false;
  const int chunks = (call.k + 127) / 128;
  const int waves = chunks >= 8 ? 8 : chunks >= 4 ? 4 : chunks >= 2 ? 2 : 1;
  const unsigned n = static_cast<unsigned>(blocks);
  if (int4) {
    *status = call.type == RUYAMD_DTYPE_BF16  ? LaunchStreamInt4Bf16(stream, args, n, waves, rows, cols)
              : call.type == RUYAMD_DTYPE_F16 ? LaunchStreamInt4F16(stream, args, n, waves, rows, cols)
                                              : LaunchStreamInt4F32(stream, args, n, waves, rows, cols);
  } else {
    *status = call.type == RUYAMD_DTYPE_BF16  ? LaunchStreamType<false, RUYAMD_DTYPE_BF16>(stream, args, n, waves, rows, cols)
              : call.type == RUYAMD_DTYPE_F16 ? LaunchStreamType<false, RUYAMD_DTYPE_F16>(stream, args, n, waves, rows, cols)
                                              : LaunchStreamType<false, RUYAMD_DTYPE_F32>(stream, args, n, waves, rows, cols);
  }
  return true;
}

}  // namespace grouped
}  // namespace ruyamd
