// Products of 4-bit values on tiles of 256x256, four waves of 128x128, one to a SIMD.
//
// A fragment of 16 bytes to a lane, a step of 128 bytes of every row and a wave of 8 x 8 blocks of 16x16 are what the largest tile
// of 8-bit integers has too, and the instructions take as long; so the steps run on the same schedule
// (paired_schedule.h): which blocks an instruction multiplies, when a fragment's registers take their next value from
// LDS, when the loads of the step after the next go out and where the barriers stand. Accumulators are in the second register
// file, and instructions are written out, for the reasons that int8_traits.h gives.
//
// What is added here is the scales. Those of a pair of steps are 16 bytes of a row. They come to LDS as they lie,
// and each lane reads the rows that it loaded itself, transposes them (mxfp4_device.h) and writes them back to where all
// waves read them, one word to a fragment of either half of either step. A fragment's word is read when the fragment of
// a pair's first step is, into the register of the word before: it is free, and wanted, when the fragment's registers are.
//   odd step 2 S - 1, behind its last loads: the scales of pair S + 1 go out to LDS (kRaw);
//   even step 2 S, behind barrier 2, which has waited for them: each lane reads its rows;
//   odd step 2 S + 1, in front of barrier 1: and writes them, transposed (kScales: pair S has been read by all waves
//     in front of barrier 2 of the even step). The words of pair S + 1 are read behind barrier 2 of this step, and in front of
//     barrier 2 of the next.
//
// Tiles left after full rounds of all CUs, a quarter of a round or less, are made as quarters of 128x128 by four workgroups each
// (mxfp4_tile.h, four stages): 4352 x 4096 x 2048, 272 tiles, 38.3 -> 33 us; 5120 x 4096 x 8192, 320 tiles, 104 -> 87. Of half a round two rounds of
// quarters take longer than one of whole tiles (6144 x 4096 x 2048 44.5 us and 38.9).
//
// 8192 x 8192 x 8192: 238 to 261 us on most cards, 4.2 to 4.6 PFLOP/s (285 on one, of uniformly random bytes); a loop of these instructions
// alone (ruyamd_diag_mfma_ceiling), on random values in registers, makes 7.7 to 7.8 and on zeros 9.7. What bounds it is the power that the
// card may take: it runs at 1.9 of its 2.4 GHz with the matrix cores busy in 57 % of the cycles, over a deeper
// product (4096 x 4096 x 32768, 5.1 PFLOP/s) at 1.7 to 1.8 with 66 to 68 %; LDS has bank conflicts in 17 % of its own cycles. What a tile
// costs beside its steps of 256 (`more` in kTiles, mxfp4_gemm.hip: its first loads and its write-back) bounds shallow products: 8 experts of
// 4096 x 2048 and 8192 tokens, 8 steps to a tile, 62 us where expert i has a share of (i + 1) ^ -0.5, 2.2 PFLOP/s at 2.4 GHz with the matrix
// cores busy in 24 % of the cycles; 53 where all have one share, which leaves no part of a round.
#include "mxfp4_large.h"
#include "mxfp4_tile.h"
#include "paired_schedule.h"

namespace ruyamd {
namespace mxfp4 {
namespace {

namespace ps = paired_schedule;

constexpr int kTile = 256, kStepBytes = 128;
constexpr int kSide = kTile * kStepBytes, kStage = 2 * kSide;  // bytes in LDS: of a side's step, of a step
constexpr int kRaw = 2 * kStage, kScales = kRaw + 2 * kTile * 16, kFifths = kScales + 2 * kTile * 16;
constexpr int kLds = kFifths + 2 * kTile * 4;
static_assert(4 * WriteBack<ps::kBlocks, ps::kBlocks>::kLds <= kLds, "");
static_assert(4 * (256 * kStepBytes) + 256 * 16 + 2 * (256 * 20) <= kLds && kLds <= 160 << 10, "a quarter's four stages, its scales and two pairs of them as they lie");
static_assert(ps::kBlocks == 8 && ps::kWaves == 4 && ps::kLoads * ps::kRowsPerLoad * ps::kWaves == kTile, "");

// The instruction with byte kByte of either side's scales. (The compiler's hazard checks do not look inside: an
// accumulator is touched by nothing else between the first of these and Drain.)
#define RUYAMD_MX_MMA(bytes)                                                                               \
  if constexpr (kFirst)                                                                                    \
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 " bytes " cbsz:4 blgp:4"         \
                 : "=a"(acc)                                                                               \
                 : "v"(a), "v"(b), "v"(a_scale), "v"(b_scale));                                            \
  else                                                                                                     \
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " bytes " cbsz:4 blgp:4"        \
                 : "+a"(acc)                                                                               \
                 : "v"(a), "v"(b), "v"(a_scale), "v"(b_scale))
template <int kByte, bool kFirst>
__device__ __forceinline__ void TiedMma(const v4i& a, const v4i& b, int a_scale, int b_scale, v4f& acc) {
  if constexpr (kByte == 0) {
    RUYAMD_MX_MMA("op_sel_hi:[0,0,0]");
  } else if constexpr (kByte == 1) {
    RUYAMD_MX_MMA("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  } else if constexpr (kByte == 2) {
    RUYAMD_MX_MMA("op_sel_hi:[1,1,0]");
  } else {
    RUYAMD_MX_MMA("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
  }
}
#undef RUYAMD_MX_MMA
__device__ __forceinline__ void Drain() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// A load's target, and the load, apart: M0 is written one wait state ahead of the load that uses it.
__device__ __forceinline__ void SetTarget(uint32_t lds) { asm volatile("s_mov_b32 m0, %0" : : "s"(lds)); }
template <uint32_t kOffset>
__device__ __forceinline__ void SetTargetAt(uint32_t lds) {
  asm volatile("s_add_u32 m0, %0, %1" : : "s"(lds), "n"(kOffset) : "scc");
}
__device__ __forceinline__ void LoadToTarget(uint32_t voffset, uint32_t soffset, v4i rsrc) {
  asm volatile("buffer_load_dwordx4 %0, %1, %2 offen lds" : : "v"(voffset), "s"(rsrc), "s"(soffset) : "memory");
}

// Where granule g of a side's row lies in its step: in slot g ^ Key. Rows of the M side are read so that a lane's
// accumulators of two blocks are of 8 consecutive ones, as in TileSide of grouped_gemm.h.
template <bool kM>
__device__ __forceinline__ int Key(int r) {
  return kM ? ((r >> 1) & 1) | ((r >> 3) & 3) << 1 : (r >> 1) & 7;
}
template <bool kM>
__device__ __forceinline__ constexpr int RowOfBlock(int b) {
  return kM ? (b >> 1) * 32 + (b & 1) * 4 : b * 16;
}

template <bool kWords>
__global__ __launch_bounds__(256, 1) void MxFp4LargeKernel(MulCall c) {
  using Scaling = ScaleRows<kWords>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave_m = wave >> 1, wave_n = wave & 1;
  const int tiles_m = (c.m + kTile - 1) / kTile;
  TileOf tile;
  Range range;
  int quarter;
  if (!FindTile(c.offsets, c.groups, c.n, kTile, tiles_m, &tile, &range, TilesAtOnce(c.compute_units), &quarter)) return;
  if (quarter >= 0) {
    tile.m = 2 * tile.m + (quarter & 1);
    tile.n = 2 * tile.n + (quarter >> 1);
    if (tile.m * 128 >= c.m || tile.n * 128 >= range.count) return;
    return MultiplyTile<2, 2, 4, 4, true, 4, kWords ? ScaleLoads::kAheadWords : ScaleLoads::kAhead>(c, tile, range, lds);
  }
  const int m0 = tile.m * kTile, n0 = tile.n * kTile;
  const int here_m = min(kTile, c.m - m0), here_n = min(kTile, range.count - n0);
  const int steps = (c.k + kStep - 1) / kStep, row_scales = c.k / kBlock;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  // The loads of the operands: eight of eight rows to a wave and side. (Rows past the tile's sides are the last one.)
  const v4i a_rsrc = Resource(reinterpret_cast<const char*>(c.lhs.data) + tile.group * c.lhs.matrix_bytes + m0 * c.lhs.row_bytes);
  const v4i b_rsrc = Resource(reinterpret_cast<const char*>(c.rhs.data) + (int64_t(range.begin) + n0) * c.rhs.row_bytes);
  uint32_t a_off[ps::kLoads], b_off[ps::kLoads];
  const auto granule_of = [&](auto is_m, int load) __attribute__((always_inline)) {
    return (lane & 7) ^ Key<decltype(is_m)::value>(ps::FirstRowOfLoad(wave, load) + (lane >> 3));
  };
  using IsM = std::true_type;
  using IsN = std::false_type;
#pragma unroll
  for (int i = 0; i < ps::kLoads; ++i) {
    const int r = ps::FirstRowOfLoad(wave, i) + (lane >> 3);
    a_off[i] = static_cast<uint32_t>(min(r, here_m - 1) * c.lhs.row_bytes) + granule_of(IsM(), i) * 16;
    b_off[i] = static_cast<uint32_t>(min(r, here_n - 1) * c.rhs.row_bytes) + granule_of(IsN(), i) * 16;
  }
  // Of the scales: waves 0 and 1 have those of the M side, 2 and 3 those of the N side, 64 rows to a load.
  const bool of_m = wave < 2;
  const uint8_t* const scales_base = of_m ? c.lhs.scales + tile.group * c.lhs.scales_matrix_stride + m0 * c.lhs.scale_stride
                                          : c.rhs.scales + (int64_t(range.begin) + n0) * c.rhs.scale_stride;
  const auto rows_of = [&](int i) __attribute__((always_inline)) {
    const int r = (wave & 1) * 128 + i * 64 + lane;
    return Scaling(scales_base, of_m ? min(r, here_m - 1) * c.lhs.scale_stride : min(r, here_n - 1) * c.rhs.scale_stride);
  };
  const Scaling scale_rows[2] = {rows_of(0), rows_of(1)};
  const uint32_t raw_target = __builtin_amdgcn_readfirstlane(lds_base + kRaw + wave * 2048);
  const uint32_t words_target = __builtin_amdgcn_readfirstlane(lds_base + kFifths + wave * 512);
  const auto load_scales = [&](int pair, int i) __attribute__((always_inline)) {
    scale_rows[i].Load(raw_target + i * 1024, words_target + i * 256, pair * 16, row_scales);
  };
  char* const mine = lds + kRaw + wave * 2048 + lane * 16;  // (and 1024 bytes behind that)
  struct Raw {
    v4i x;
    int fifth;
  };
  const auto read_raw = [&](int i) __attribute__((always_inline)) {
    Raw raw = {*reinterpret_cast<const v4i*>(mine + i * 1024), 0};
    if constexpr (kWords) raw.fifth = *reinterpret_cast<const int*>(lds + kFifths + wave * 512 + i * 256 + lane * 4);
    return raw;
  };
  const auto put_scales = [&](const Raw& raw, int pair, int i) __attribute__((always_inline)) {
    *reinterpret_cast<v4i*>(mine + (kScales - kRaw) + i * 1024) =
        Transposed(Scaling::Place(raw.x, raw.fifth, scale_rows[i].at, pair * 16, row_scales));
  };

  // The fragments and their scales: of the M side's rows and the N side's columns, both depth halves of a step.
  v4i fa[2][ps::kBlocks], fb[2][ps::kBlocks];
  int sa[ps::kBlocks], sb[ps::kBlocks];
  v4f acc[ps::kBlocks][ps::kBlocks];
  const int a_row = wave_m * 128 + (l >> 2) * 8 + (l & 3), b_row = wave_n * 128 + l;
  int a_at[2], b_at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    a_at[h] = a_row * kStepBytes + (((h * 4 + q) ^ Key<true>(a_row)) << 4);
    b_at[h] = kSide + b_row * kStepBytes + (((h * 4 + q) ^ Key<false>(b_row)) << 4);
  }
  const char* const a_scales = lds + kScales + a_row * 16 + q * 4;
  const char* const b_scales = lds + kScales + (kTile + b_row) * 16 + q * 4;
  const auto read_a = [&](int slot, int h, int i) __attribute__((always_inline)) {
    fa[h][i] = *reinterpret_cast<const v4i*>(lds + slot * kStage + a_at[h] + RowOfBlock<true>(i) * kStepBytes);
    if (slot == 0 && h == 0) sa[i] = *reinterpret_cast<const int*>(a_scales + RowOfBlock<true>(i) * 16);
  };
  const auto read_b = [&](int slot, int h, int j) __attribute__((always_inline)) {
    fb[h][j] = *reinterpret_cast<const v4i*>(lds + slot * kStage + b_at[h] + RowOfBlock<false>(j) * kStepBytes);
    if (slot == 0 && h == 0) sb[j] = *reinterpret_cast<const int*>(b_scales + RowOfBlock<false>(j) * 16);
  };

  // A load of step s (any: zeros past the depth) into its slot.
  const uint32_t targets = __builtin_amdgcn_readfirstlane(lds_base + wave * ps::kLoads * 1024);
  const auto issue = [&](int s, auto is_m, int i) __attribute__((always_inline)) {
    constexpr bool kIsM = decltype(is_m)::value;
    const int left = (c.k - s * kStep) / kBlock;  // granules
    SetTarget(targets + (s & 1) * kStage + (kIsM ? 0 : kSide) + i * 1024);
    asm volatile("s_nop 0");
    const uint32_t off = granule_of(is_m, i) < left ? (kIsM ? a_off[i] : b_off[i]) : kNothing;
    LoadToTarget(off, static_cast<uint32_t>(s) * kStepBytes, kIsM ? a_rsrc : b_rsrc);
  };

  load_scales(0, 0);
  load_scales(0, 1);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int i = 0; i < ps::kLoads; ++i) issue(s, IsN(), i);
#pragma unroll
    for (int i = 0; i < ps::kLoads; ++i) issue(s, IsM(), i);
  }
  WaitVmcnt<4 * ps::kLoads>();
  Raw raw[2] = {read_raw(0), read_raw(1)};
  put_scales(raw[0], 0, 0);
  put_scales(raw[1], 0, 1);
  // (What has been read of kRaw is in registers: put_scales has used it.)
  load_scales(1, 0);
  load_scales(1, 1);
  WaitVmcnt<2 * ps::kLoads + 2 * Scaling::kLoads>();
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < ps::kRowsReadAhead; ++i) read_a(0, h, i);
#pragma unroll
    for (int p = 0; p < ps::kColumnsReadAhead; ++p) read_b(0, h, ps::ColumnAt(0, 0, p));
  }

  const auto step = [&](int s, auto parity, auto full, auto first) __attribute__((always_inline)) {
    constexpr int kParity = decltype(parity)::value;  // of s, hence the slot
    constexpr bool kFull = decltype(full)::value;
    uint32_t refill = static_cast<uint32_t>(s + 2) * kStepBytes;
    if constexpr (kFull) asm volatile("" : "+s"(refill));
    StaticFor<ps::kInstructions>([&](auto number) __attribute__((always_inline)) {
      constexpr int n = decltype(number)::value;
      constexpr ps::Mma mma = ps::MmaAt(kParity, n);
      if constexpr (n == ps::kTiming.barrier1) __syncthreads();
      if constexpr (n == ps::kTiming.barrier2) {
        WaitVmcnt<ps::kTiming.loads_left_at_barrier2>();
        __syncthreads();
      }
      __builtin_amdgcn_sched_barrier(0);
      TiedMma<2 * kParity + mma.half, decltype(first)::value && mma.half == 0>(fa[mma.half][mma.row], fb[mma.half][mma.col],
                                                                               sa[mma.row], sb[mma.col], acc[mma.row][mma.col]);
      __builtin_amdgcn_sched_barrier(0);
      constexpr ps::Read read = ps::ReadBehind(kParity, n);
      if constexpr (read.valid) {
        constexpr int slot = read.of_next_step ? kParity ^ 1 : kParity;
        if constexpr (read.is_a)
          read_a(slot, read.half, read.index);
        else
          read_b(slot, read.half, read.index);
      }
      constexpr ps::Load target = ps::LoadBehind(n + 1), load = ps::LoadBehind(n);
      if constexpr (kFull && target.valid)
        SetTargetAt<uint32_t(kParity * kStage + (target.is_b ? kSide : 0) + target.index * 1024)>(targets);
      if constexpr (load.valid) {
        if constexpr (kFull)
          LoadToTarget(load.is_b ? b_off[load.index] : a_off[load.index], refill, load.is_b ? b_rsrc : a_rsrc);
        else
          issue(s + 2, std::integral_constant<bool, !load.is_b>(), load.index);
      }
      // The scales. (Where nothing else stands.)
      if constexpr (kParity == 0 && (n == 112 || n == 116)) raw[(n - 112) / 4] = read_raw((n - 112) / 4);
      if constexpr (kParity == 1 && (n == 3 || n == 13)) put_scales(raw[n / 13], (s + 1) / 2, n / 13);
      if constexpr (kParity == 1 && (n == 118 || n == 122)) load_scales((s + 3) / 2, (n - 118) / 4);
    });
    __builtin_amdgcn_sched_barrier(0);
  };
  using Even = std::integral_constant<int, 0>;
  using Odd = std::integral_constant<int, 1>;
  using Yes = std::true_type;
  using No = std::false_type;
  // (Straight-line loop bodies, as for 8-bit integers: with a branch on the step's parity in the loop the register
  // allocator moves accumulators through scratch memory.)
  const int full_end = c.k / kStep - 2;  // steps whose loads lie inside the depth
  if (full_end > 0)
    step(0, Even(), Yes(), Yes());
  else
    step(0, Even(), No(), Yes());
  int s = 1;
  for (; s + 1 < full_end; s += 2) {
    step(s, Odd(), Yes(), No());
    step(s + 1, Even(), Yes(), No());
  }
  for (; s + 1 < steps; s += 2) {
    step(s, Odd(), No(), No());
    step(s + 1, Even(), No(), No());
  }
  if (s < steps) step(s, Odd(), No(), No());
  Drain();
  WaitVmcnt<0>();

  // (LDS is the write-back's now.)
  __syncthreads();
  using Out = WriteBack<ps::kBlocks, ps::kBlocks>;
  Out{c, acc, lds + wave * Out::kLds, c.bias ? c.bias + tile.group * c.bias_stride + m0 + wave_m * 128 : nullptr,
      m0 + wave_m * 128, int64_t(range.begin) + n0 + wave_n * 128, here_m - wave_m * 128, here_n - wave_n * 128}();
}

template <bool kWords>
hipError_t Launch(hipStream_t stream, const MulCall& call, unsigned blocks) {
  static const hipError_t attribute =
      hipFuncSetAttribute(reinterpret_cast<const void*>(&MxFp4LargeKernel<kWords>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (attribute != hipSuccess) return attribute;
  hipLaunchKernelGGL(MxFp4LargeKernel<kWords>, dim3(blocks), dim3(256), kLds, stream, call);
  return hipGetLastError();
}

}  // namespace

hipError_t LaunchLarge(hipStream_t stream, const MulCall& call, unsigned blocks) {
  return ScalesNeedWords(call) ? Launch<true>(stream, call, blocks) : Launch<false>(stream, call, blocks);
}

}  // namespace mxfp4
}  // namespace ruyamd
