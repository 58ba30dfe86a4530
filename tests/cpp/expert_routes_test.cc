// What the calls for layers of experts launch, on the model of the HIP runtime
// in runtime_model_test.cc (no operand is touched, no device needed). Reads
// calls from the standard input, a line each:
//
//   sort <type of the numbers> <tokens> <top> <count>
//   mxfp4 <type of dst> <order of dst> <rows> <columns> <depth> <groups, 0: none>
//       <bytes of a row of lhs> <scales of one> <bytes of a matrix of lhs> <scales of one>
//       <bytes of a row of rhs> <scales of one> <address of the first bytes modulo 16> <forced tile: three numbers>
//
// and answers each with a line of the call's result and the kernels' names.
#define main runtime_model_main
#include "runtime_model_test.cc"
#undef main

namespace {

char* Memory(int i) {
  static const std::size_t room = std::size_t(1) << 38;
  static char* const at = [] {
    void* const p = mmap(nullptr, 4 * room, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
    if (p == MAP_FAILED) std::abort();
    R().device[static_cast<char*>(p)] = 4 * room;
    return static_cast<char*>(p);
  }();
  return at + i * room;
}

int Sort(ruyamd_ctx* ctx) {
  int type, tokens, top, count;
  if (std::scanf("%d %d %d %d", &type, &tokens, &top, &count) != 4) std::abort();
  const ruyamd_mat experts = Mat(type, Memory(0), top, tokens, RUYAMD_ORDER_COL_MAJOR);
  ruyamd_routing routing = {};
  routing.offsets = reinterpret_cast<int32_t*>(Memory(1));
  routing.places = reinterpret_cast<int32_t*>(Memory(2));
  routing.sources = reinterpret_cast<int32_t*>(Memory(3));
  routing.tokens = tokens;
  routing.top = top;
  routing.count = count;
  return ruyamd_sort_tokens(ctx, &experts, &routing);
}

int MulMxFp4(ruyamd_ctx* ctx) {
  int type, order, m, n, k, count, address, tile[3];
  ruyamd_mxfp4_mat lhs = {}, rhs = {};
  long long bytes, scales;
  if (std::scanf("%d %d %d %d %d %d %d %d %lld %lld %d %d %d %d %d %d", &type, &order, &m, &n, &k, &count, &lhs.row_bytes,
                 &lhs.scale_stride, &bytes, &scales, &rhs.row_bytes, &rhs.scale_stride, &address, &tile[0], &tile[1],
                 &tile[2]) != 16)
    std::abort();
  lhs.data = Memory(0) + address;
  lhs.scales = reinterpret_cast<uint8_t*>(Memory(1) + address);
  lhs.rows = m;
  lhs.matrix_bytes = bytes;
  lhs.scales_matrix_stride = scales;
  rhs.data = Memory(2) + address;
  rhs.scales = reinterpret_cast<uint8_t*>(Memory(3) + address);
  rhs.rows = n;
  lhs.cols = rhs.cols = k;
  const ruyamd_mat dst = Mat(type, Memory(3) + (std::size_t(1) << 37), m, n, order);
  ruyamd_mul_params params = Params(RUYAMD_DTYPE_F32);
  ruyamd_groups groups = {};
  groups.offsets = reinterpret_cast<int32_t*>(Memory(1) + (std::size_t(1) << 37));
  groups.count = count;
  if (ruyamd_ctx_force_tile(ctx, tile[0], tile[1], tile[2]) != RUYAMD_OK) std::abort();
  return ruyamd_mul_mxfp4(ctx, &lhs, &rhs, count ? &groups : nullptr, &params, &dst);
}

}  // namespace

int main() {
  R().fill_allocations = false;
  Context c;
  char what[32];
  while (std::scanf("%31s", what) == 1) {
    R().log.clear();
    const int rc = std::strcmp(what, "sort") == 0 ? Sort(c.ctx) : MulMxFp4(c.ctx);
    std::printf("%d", rc);
    for (const std::string& kernel : R().log) std::printf(" %s", kernel.c_str());
    std::printf("\n");
  }
  return 0;
}
