// Launches of the tiled kernel of grouped products.
#include "grouped_gemm.h"

namespace ruyamd {
namespace grouped {
namespace {

template <int kType, Runs kRunsM, Runs kRunsN, bool kDirect>
void LaunchOne(hipStream_t stream, const GemmArgs& args, unsigned blocks) {
  hipLaunchKernelGGL((GroupedGemmKernel<kType, kRunsM, kRunsN, 2, 2, 4, 4, kDirect>), dim3(blocks), dim3(256), 0, stream,
                     args);
}

template <int kType, bool kDirect>
void LaunchRuns(hipStream_t stream, const GemmArgs& args, Runs m, Runs n, unsigned blocks) {
  if (m == Runs::kPlain && n == Runs::kPlain) return LaunchOne<kType, Runs::kPlain, Runs::kPlain, kDirect>(stream, args, blocks);
  if (m == Runs::kPlain) return LaunchOne<kType, Runs::kPlain, Runs::kAcross, kDirect>(stream, args, blocks);
  if (n == Runs::kPlain) return LaunchOne<kType, Runs::kAcross, Runs::kPlain, kDirect>(stream, args, blocks);
  LaunchOne<kType, Runs::kAcross, Runs::kAcross, kDirect>(stream, args, blocks);
}

template <bool kDirect>
void LaunchType(hipStream_t stream, const GemmArgs& args, int type, Runs m, Runs n, unsigned blocks) {
  if (type == RUYAMD_DTYPE_BF16) return LaunchRuns<RUYAMD_DTYPE_BF16, kDirect>(stream, args, m, n, blocks);
  if (type == RUYAMD_DTYPE_F16) return LaunchRuns<RUYAMD_DTYPE_F16, kDirect>(stream, args, m, n, blocks);
  LaunchRuns<RUYAMD_DTYPE_F32, kDirect>(stream, args, m, n, blocks);
}

}  // namespace

bool LaunchTiles(hipStream_t stream, const Call& call, hipError_t* status) {
  constexpr int kTile = 128;
  const int bytes = call.type == RUYAMD_DTYPE_F32 ? 4 : 2, granule = 16 / bytes;
  const bool columns = call.dealt == Dealt::kColumns;
  // The M side is the one along which dst is contiguous. (Columns that are dealt
  // to groups stay on the N side; a dst by rows is then written value by value.)
  const bool swapped = !columns && call.dst_rs != 1;
  GemmArgs a;
  a.dealt = call.dealt;
  a.depth = call.k;
  a.offsets = call.offsets;
  a.groups = call.groups;
  a.bias = call.bias;
  a.bias_stride = call.bias_stride;
  a.clamp_min = call.clamp_min;
  a.clamp_max = call.clamp_max;
  a.dst = call.dst;
  a.dst_f32 = call.dst_type == RUYAMD_DTYPE_F32;
  a.dst_group_stride = columns ? 0 : call.matrix_stride;
  const auto side = [&](bool lhs, Side* s) {
    const int64_t along = lhs ? call.lhs_rs : call.rhs_cs, depth = lhs ? call.lhs_cs : call.rhs_rs;
    s->data = lhs ? call.lhs : call.rhs;
    s->count = lhs ? call.m : call.n;
    s->group_stride = columns && lhs ? call.matrix_stride : 0;
    // (A side of one row, or a depth of one, has both strides 1: either order will do.)
    const Runs runs = depth == 1 ? Runs::kPlain : Runs::kAcross;
    s->pitch = runs == Runs::kPlain ? along : depth;
    return runs;
  };
  const Runs runs_m = side(!swapped, &a.m), runs_n = side(swapped, &a.n);
  a.dst_m_stride = swapped ? call.dst_cs : call.dst_rs;
  a.dst_n_stride = swapped ? call.dst_rs : call.dst_cs;

  // Offsets inside a tile are 31 bits.
  if (a.m.pitch > (int64_t(1) << 31) / (bytes * kTile) - 128 || a.n.pitch > (int64_t(1) << 31) / (bytes * kTile) - 128)
    return false;
  const auto aligned = [&](const Side& s, Runs runs, bool dealt_rows) {
    if (reinterpret_cast<uintptr_t>(s.data) % 16 || s.pitch % granule || s.group_stride % granule) return false;
    // Runs along the depth end and, where it is dealt, begin anywhere.
    if (runs == Runs::kPlain) return columns && call.k % granule == 0;
    return !(columns && dealt_rows) && s.count % granule == 0;
  };
  const bool direct = aligned(a.m, runs_m, false) && aligned(a.n, runs_n, true);
  const int dst_bytes = a.dst_f32 ? 4 : 2;
  a.vector_stores = a.dst_m_stride == 1 && reinterpret_cast<uintptr_t>(a.dst) % (4 * dst_bytes) == 0 &&
                    a.dst_n_stride % 4 == 0 && a.dst_group_stride % 4 == 0;

  const int64_t tiles_m = (int64_t(a.m.count) + kTile - 1) / kTile;
  const int64_t tiles_n =
      columns ? a.n.count / kTile + min(call.groups, a.n.count) : ((int64_t(a.n.count) + kTile - 1) / kTile) * call.groups;
  const int64_t blocks = (tiles_m * tiles_n + 7) / 8 * 8;
  if (blocks > 0x7fffffff) return false;
  if (direct)
    LaunchType<true>(stream, a, call.type, runs_m, runs_n, static_cast<unsigned>(blocks));
  else
    LaunchType<false>(stream, a, call.type, runs_m, runs_n, static_cast<unsigned>(blocks));
  *status = hipGetLastError();
  return true;
}

}  // namespace grouped
}  // namespace ruyamd
