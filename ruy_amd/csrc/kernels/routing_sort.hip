// Choices sorted by expert, keeping their order (ruyamd_sort_tokens).
//
// The place of choice i of expert e is the number of choices of experts before e plus
// the number of e's own before i: counting alone, no comparison of choices with each other, and
// no atomic whose order would show.
//
// Few choices and experts, one launch: a workgroup to an expert counts, over all choices, those of
// experts before its own and its own, and hands out places to the latter. The choices are read by every
// workgroup, out of L2 after the first. Many of either, three launches: a wave to a part of the choices counts what each expert
// has in it; one workgroup adds these up, over parts and experts; a wave to a part hands out places, 64 choices at a time, those of
// one expert among them found by comparing the numbers bit by bit over the wave. The counts of a part lie meanwhile
// where its places will be (a part has as many choices as there are experts, or more): no other memory is needed.
//
// What bounds both is latency, not the 8 to 20 bytes of a choice: a launch, a read of the choices, a sum over the workgroup and the
// writes of the places. Among 64 experts, 64-bit numbers: 32 choices 3.3 us; 32768 10.2 in one launch, whose workgroups have 2048 choices to
// a wave and read all 256 KB out of L2 (half of the time; with all 32 loads of a lane on their way at once no less); 131072 14.4 in three.
#include <algorithm>

#include "grouped_gemm.h"
#include "launch_geometry.h"
#include "routing.h"

namespace ruyamd {
namespace routing {
namespace {

// What stands for the expert of a choice that has none, and for that of a choice behind the last.
constexpr uint32_t kNone = 0xffffffffu, kPast = 0xfffffffeu;

// The expert of choice i, or kNone.
template <bool kWide, bool kPlain>
__device__ __forceinline__ uint32_t NumberOf(const SortCall& c, int64_t i) {
  int64_t at = i;
  if constexpr (!kPlain) {
    const int t = static_cast<int>(uint32_t(i) / uint32_t(c.top));
    at = t * c.cs + (i - int64_t(t) * c.top) * c.rs;
  }
  if constexpr (kWide) {
    const uint2 v = static_cast<const uint2*>(c.experts)[at];
    return v.y == 0 && v.x < uint32_t(c.count) ? v.x : kNone;
  } else {
    const uint32_t v = static_cast<const uint32_t*>(c.experts)[at];
    return v < uint32_t(c.count) ? v : kNone;
  }
}
// Those of the lane in kAtOnce rows of 64 from `at` on, of choices in front of `end`.
constexpr int kAtOnce = 8;
template <bool kWide, bool kPlain>
__device__ __forceinline__ void NumbersOf(const SortCall& c, int64_t at, int64_t end, int lane, uint32_t (&v)[kAtOnce]) {
  if (at + 64 * kAtOnce <= end) {
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) v[u] = NumberOf<kWide, kPlain>(c, at + lane + u * 64);
  } else {
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int64_t mine = at + lane + u * 64;
      v[u] = NumberOf<kWide, kPlain>(c, min(mine, end - 1));
      if (mine >= end) v[u] = kPast;
    }
  }
}

__device__ __forceinline__ int BelowMe(uint64_t lanes) {
  return __builtin_amdgcn_mbcnt_hi(uint32_t(lanes >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(lanes), 0));
}

__device__ __forceinline__ int WaveSum(int v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

constexpr int kMostWaves = 16;
constexpr int kHeld = 32 * 64;  // choices that a wave looks at before it counts on, a bit of each lane to each 64

// Expert blockIdx.x; every wave has a contiguous part of the choices.
template <bool kWide, bool kPlain>
__global__ __launch_bounds__(64 * kMostWaves) void SortByExpertKernel(SortCall c) {
  __shared__ int lower[kMostWaves], own[kMostWaves];
  const int waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = c.tokens * c.top, expert = blockIdx.x;
  const int64_t part = (int64_t(n) + 64 * waves - 1) / (64 * waves) * 64;
  const int64_t begin = wave * part, end = min(int64_t(n), begin + part);
  // Which of the lane's 32 choices of kHeld from `at` on are the expert's. first: the first time that they are looked at.
  int lower_here = 0, own_here = 0;
  const auto look = [&](int64_t at, bool first) __attribute__((always_inline)) -> uint32_t {
    uint32_t held = 0;
#pragma unroll
    for (int b = 0; b < 32 / kAtOnce; ++b) {
      const int64_t from = at + b * (64 * kAtOnce);
      if (from >= end) break;
      uint32_t v[kAtOnce];
      NumbersOf<kWide, kPlain>(c, from, end, lane, v);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        held |= uint32_t(v[u] == uint32_t(expert)) << (b * kAtOnce + u);
        if (!first) continue;
        lower_here += v[u] < uint32_t(expert);
        if (expert == 0 && v[u] == kNone) c.places[from + u * 64 + lane] = -1;
      }
    }
    if (first) own_here += __builtin_popcount(held);
    return held;
  };
  const uint32_t first_held = look(begin, true);
  for (int64_t at = begin + kHeld; at < end; at += kHeld) look(at, true);
  lower_here = WaveSum(lower_here);
  own_here = WaveSum(own_here);
  if (lane == 0) {
    lower[wave] = lower_here;
    own[wave] = own_here;
  }
  __syncthreads();
  int first = 0, next = 0, total = 0;
  for (int w = 0; w < waves; ++w) {
    first += lower[w];
    next += w < wave ? own[w] : 0;
    total += own[w];
  }
  if (threadIdx.x == 0) {
    c.offsets[expert] = first;
    if (expert == c.count - 1) c.offsets[c.count] = first + total;
  }
  if (expert == c.count - 1 && c.sources)
    for (int64_t p = int64_t(first) + total + threadIdx.x; p < n; p += blockDim.x) c.sources[p] = -1;
  next = __builtin_amdgcn_readfirstlane(next + first);
  for (int64_t at = begin; at < end; at += kHeld) {
    uint32_t held = at == begin ? first_held : look(at, false);
    // Lane i has, of the 64 choices number i, which are the expert's and how many places are taken before them. A
    // lane then goes through its own choices only: few, where there are many experts.
    uint32_t low = 0, high = 0;
#pragma unroll
    for (int b = 0; b < 32 / kAtOnce; ++b) {
      if (at + b * (64 * kAtOnce) >= end) break;
#pragma unroll
      for (int i = b * kAtOnce; i < (b + 1) * kAtOnce; ++i) {
        const uint64_t all = __ballot(held >> i & 1);
        low = lane == i ? static_cast<uint32_t>(all) : low;
        high = lane == i ? static_cast<uint32_t>(all >> 32) : high;
      }
    }
    const int here = __builtin_popcount(low) + __builtin_popcount(high), upto = grouped::InclusiveSum(here);
    const int before = next + upto - here;
    next += __builtin_amdgcn_readlane(upto, 63);
    while (__any(held != 0)) {
      const int i = held ? __builtin_ctz(held) : 0;
      const uint32_t l = __shfl(low, i), h = __shfl(high, i);
      const int place = __builtin_amdgcn_mbcnt_hi(h, __builtin_amdgcn_mbcnt_lo(l, __shfl(before, i)));
      if (held) {
        const int64_t mine = at + i * 64 + lane;
        c.places[mine] = place;
        if (c.sources) c.sources[place] = static_cast<int>(mine);
      }
      held &= held - 1;
    }
  }
}

// Part b: choices b * part .. and, of the last of `parts`, all behind them.
struct Parts {
  int part, parts;
};
__device__ __forceinline__ int EndOf(const Parts& p, int b, int n) { return b == p.parts - 1 ? n : (b + 1) * p.part; }

template <bool kWide, bool kPlain>
__global__ __launch_bounds__(64) void CountKernel(SortCall c, Parts parts) {
  extern __shared__ int counts[];
  const int lane = threadIdx.x, begin = blockIdx.x * parts.part, end = EndOf(parts, blockIdx.x, c.tokens * c.top);
  for (int e = lane; e < c.count; e += 64) counts[e] = 0;
  __syncthreads();
  for (int64_t at = begin; at < end; at += 64 * kAtOnce) {
    uint32_t v[kAtOnce];
    NumbersOf<kWide, kPlain>(c, at, end, lane, v);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      if (v[u] < kPast) atomicAdd(&counts[v[u]], 1);  // (a sum of ones: any order)
  }
  __syncthreads();
  for (int e = lane; e < c.count; e += 64) c.places[begin + e] = counts[e];
}

// One workgroup: counts to the sums of the counts of the parts before, and the offsets. 1024
// threads are `across` experts (a power of two, as many as there are or more, or all of them) by 1024 / across runs of the parts.
__global__ __launch_bounds__(1024) void AddUpKernel(SortCall c, Parts parts, int across) {
  __shared__ int sums[1024], waves[16];
  const int runs = 1024 / across, e0 = threadIdx.x & (across - 1), run = threadIdx.x / across, lane = threadIdx.x & 63;
  const int length = (parts.parts + runs - 1) / runs;
  const int from = min(run * length, parts.parts), to = min(from + length, parts.parts);
  int before = 0;  // places of all experts so far
  for (int base = 0; base < c.count; base += across) {
    const int e = base + e0;
    int sum = 0;
    if (e < c.count) {
#pragma unroll 8
      for (int b = from; b < to; ++b) sum += c.places[b * parts.part + e];
    }
    sums[threadIdx.x] = sum;
    __syncthreads();
    int first = 0, all = 0;
    for (int r = 0; r < runs; ++r) {
      const int s = sums[r * across + e0];
      first += r < run ? s : 0;
      all += s;
    }
    if (e < c.count) {
#pragma unroll 8
      for (int b = from; b < to; ++b) {
        int32_t* const at = &c.places[b * parts.part + e];
        const int count = *at;
        *at = first;
        first += count;
      }
    }
    // Of the experts of this round, in order: the threads of the first run.
    int upto = run == 0 ? all : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    if (lane == 63) waves[threadIdx.x >> 6] = upto;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < int(threadIdx.x >> 6)) upto += waves[w];
      total += waves[w];
    }
    if (run == 0 && e < c.count) c.offsets[e] = before + upto - all;
    before += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) c.offsets[c.count] = before;
}

template <bool kWide, bool kPlain>
__global__ __launch_bounds__(64) void PlaceKernel(SortCall c, Parts parts, int bits) {
  extern __shared__ int counts[];
  volatile int* const next = counts;
  const int lane = threadIdx.x, n = c.tokens * c.top;
  const int begin = blockIdx.x * parts.part, end = EndOf(parts, blockIdx.x, n);
  for (int e = lane; e < c.count; e += 64) next[e] = c.offsets[e] + c.places[begin + e];
  __syncthreads();
  const int used = c.offsets[c.count];
  for (int64_t at = begin; at < end; at += 64) {
    const int64_t mine = at + lane;
    const uint32_t v = mine < end ? NumberOf<kWide, kPlain>(c, mine) : kPast;
    uint64_t same = __ballot(v < kPast);
    for (int bit = 0; bit < bits; ++bit) {
      const bool set = v >> bit & 1;
      const uint64_t with = __ballot(set);
      same &= set ? with : ~with;
    }
    int place = -1;
    if (v < kPast) {
      const int rank = BelowMe(same);
      place = next[v] + rank;
      __builtin_amdgcn_wave_barrier();
      if (rank == __builtin_popcountll(same) - 1) next[v] = place + 1;
    }
    __builtin_amdgcn_wave_barrier();
    if (mine < end) {
      c.places[mine] = place;
      if (c.sources) {
        if (place >= 0) c.sources[place] = static_cast<int>(mine);
        if (mine >= used) c.sources[mine] = -1;
      }
    }
  }
}

template <bool kWide, bool kPlain>
hipError_t Launch(hipStream_t stream, const SortCall& c, bool one_launch) {
  const int64_t n = int64_t(c.tokens) * c.top;
  // Parts: as long as there are experts at least, some thousand at most.
  const int64_t part = std::max<int64_t>({(c.count + 63) / 64 * 64, 512, (n + 1023) / 1024 / 64 * 64});
  // One launch reads all choices once to each expert, and a wave keeps in registers what it has seen of 2048 of them. (us, one and
  // three, int64: 32768 choices, 16 experts 10.3 and 12.9, 256 10.0 and 15.9, 512 17.2 and 20.1; 40000, 16 experts 13.3 and 13.7, 256 12.0 and
  // 17.6; 65536, 16 experts 21.4 and 13.6, 64 18.9 and 12.9, 256 18.4 and 18.4, 512 32.0 and 24.8.)
  if (one_launch || c.count > 16384 || n < 2 * part || (n <= 49152 && n * c.count <= int64_t(1) << 25)) {
    const int waves = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMostWaves, (n + 255) / 256)));
    hipLaunchKernelGGL((SortByExpertKernel<kWide, kPlain>), dim3(c.count), dim3(64 * waves), 0, stream, c);
    return hipGetLastError();
  }
  const Parts parts = {static_cast<int>(part), static_cast<int>(n / part)};
  int across = 1, bits = 0;
  while (across < c.count && across < 1024) across *= 2;
  while ((1 << bits) < c.count) ++bits;
  hipLaunchKernelGGL((CountKernel<kWide, kPlain>), dim3(parts.parts), dim3(64), c.count * 4, stream, c, parts);
  hipLaunchKernelGGL(AddUpKernel, dim3(1), dim3(1024), 0, stream, c, parts, across);
  hipLaunchKernelGGL((PlaceKernel<kWide, kPlain>), dim3(parts.parts), dim3(64), c.count * 4, stream, c, parts, bits);
  return hipGetLastError();
}

}  // namespace

hipError_t LaunchSort(hipStream_t stream, const SortCall& c, bool force_generic) {
  const bool plain = (c.rs == 1 || c.top <= 1) && (c.cs == c.top || c.tokens <= 1);
  if (c.wide) return plain ? Launch<true, true>(stream, c, force_generic) : Launch<true, false>(stream, c, force_generic);
  return plain ? Launch<false, true>(stream, c, force_generic) : Launch<false, false>(stream, c, force_generic);
}

}  // namespace routing
}  // namespace ruyamd
