// Tokens copied to their places, the rows in these places added up, and the
// gradients of that (ruyamd_dispatch_tokens, ruyamd_combine_tokens,
// ruyamd_combine_tokens_gradients).
//
// All of these go token by token: what belongs to a token once (its values, its sum, its gradient) is
// read or written once, and its rows, wherever they are, as whole lines. A lane has units of 16
// bytes (8 values of 16 bits, 4 of 32); the last unit of a row that is no whole number of them
// ends where the row ends, and overlaps the one before.
//
// All are copies with a little arithmetic, bound by HBM, and by the launch where there is little to copy. What is left to choose is how much a lane
// has on its way at once (WithUnits, and four choices of a token together) and which writes go past the caches (kStreamFrom).
// Moved, 8192 tokens of 4096 values in bfloat16 and two places each, 201 MB: to their places 33 us, 6.1 TB/s; added up, 37 us, 5.4;
// gradients, 336 MB, 70 us, 4.8, of which the rows alone would be 35. Sixteen tokens of 2048 values: 2.8 us and 3.3.
#include <algorithm>

#include "granule.h"
#include "grouped_device.h"
#include "launch_geometry.h"
#include "routing.h"

namespace ruyamd {
namespace routing {
namespace {

using granule::v4i;
using granule::v4i_unaligned;
using grouped::LoadFloat;
using grouped::RoundPair;
using grouped::StoreFloat;

constexpr int Bytes(int type) { return type == RUYAMD_DTYPE_F32 ? 4 : 2; }

// kValues values from number `at` on.
template <int kType, int kValues>
__device__ __forceinline__ void Load(const void* data, int64_t at, v4i (&raw)[kValues * Bytes(kType) / 16]) {
  const v4i_unaligned* const p =
      reinterpret_cast<const v4i_unaligned*>(static_cast<const char*>(data) + at * Bytes(kType));
#pragma unroll
  for (int i = 0; i < kValues * Bytes(kType) / 16; ++i) raw[i] = p[i];
}
template <int kType, int kValues>
__device__ __forceinline__ float Value(const v4i (&raw)[kValues * Bytes(kType) / 16], int e) {
  if constexpr (kType == RUYAMD_DTYPE_F32) {
    return __int_as_float(raw[e / 4][e % 4]);
  } else {
    const uint32_t word = static_cast<uint32_t>(raw[0][e / 2]);
    if constexpr (kType == RUYAMD_DTYPE_BF16) return __uint_as_float(e % 2 ? word & 0xffff0000u : word << 16);
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(e % 2 ? word >> 16 : word)));
  }
}
// kStreamed: past the caches, for what is more than they hold anyway (kStreamFrom).
template <bool kStreamed>
__device__ __forceinline__ void StoreGranule(v4i_unaligned* p, const v4i& x) {
  if constexpr (kStreamed)
    __builtin_nontemporal_store(x, p);
  else
    *p = x;
}
template <int kType, int kValues, bool kStreamed = false>
__device__ __forceinline__ void Store(void* data, int64_t at, const float (&v)[kValues]) {
  v4i_unaligned* const p = reinterpret_cast<v4i_unaligned*>(static_cast<char*>(data) + at * Bytes(kType));
#pragma unroll
  for (int i = 0; i < kValues * Bytes(kType) / 16; ++i) {
    v4i raw;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (kType == RUYAMD_DTYPE_F32)
        raw[e] = __float_as_int(v[i * 4 + e]);
      else
        raw[e] = RoundPair<kType>(v[2 * e], v[2 * e + 1]);
    }
    StoreGranule<kStreamed>(p + i, raw);
  }
}

// A token and which of its segments of 64 * kUnits units this wave has. (Whole waves: scalars.)
struct Piece {
  int token, segment;
};
__device__ __forceinline__ int64_t FirstPiece() {
  return int64_t(blockIdx.x) * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}
__device__ __forceinline__ int64_t PieceStride() { return int64_t(gridDim.x) * (blockDim.x >> 6); }
__device__ __forceinline__ Piece PieceOf(int64_t i, int segments) {
  const int token = static_cast<int>(i / segments);
  return {token, static_cast<int>(i - int64_t(token) * segments)};
}

// The place of choice j of a token, or -1.
__device__ __forceinline__ int PlaceOf(const Call& c, int64_t token, int j) {
  const int p = c.places[token * c.top + j];
  return p >= 0 && p < c.columns ? p : -1;
}
__device__ __forceinline__ float WeightOf(const Call& c, int64_t token, int j) {
  return c.weights.data ? LoadFloat(c.weights.data, c.weights.type, j * c.weights.rs + token * c.weights.cs) : 1.0f;
}


// ---- Tokens to their places ----

template <int kBytes, int kUnits, bool kStreamed>
__global__ __launch_bounds__(256) void DispatchKernel(Call c, int segments) {
  const int lane = threadIdx.x & 63;
  const int64_t bytes = int64_t(c.width) * kBytes, pieces = int64_t(c.tokens) * segments;
  for (int64_t i = FirstPiece(); i < pieces; i += PieceStride()) {
    const Piece piece = PieceOf(i, segments);
    const char* const from = static_cast<const char*>(c.token_side.data) + piece.token * c.token_side.cs * kBytes;
    const int64_t first = int64_t(piece.segment) * (1024 * kUnits);
    v4i held[kUnits];
    int64_t at[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      at[u] = min(first + u * 1024 + lane * 16, bytes - 16);
      if (first + u * 1024 < bytes) held[u] = *reinterpret_cast<const v4i_unaligned*>(from + at[u]);
    }
    for (int j = 0; j < c.top; ++j) {
      const int place = PlaceOf(c, piece.token, j);
      if (place < 0) continue;
      char* const to = static_cast<char*>(c.place_side.data) + place * c.place_side.cs * kBytes;
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        if (first + u * 1024 < bytes) StoreGranule<kStreamed>(reinterpret_cast<v4i_unaligned*>(to + at[u]), held[u]);
    }
  }
}

// ---- The sum of a token's rows ----

template <int kType, int kDstType, int kUnits, bool kStreamed>
__global__ __launch_bounds__(256) void CombineKernel(Call c, int segments) {
  constexpr int kValues = 16 / Bytes(kType);
  constexpr int kAtOnce = 4;  // choices of a token whose rows are on their way together
  const int lane = threadIdx.x & 63;
  const int64_t pieces = int64_t(c.tokens) * segments;
  for (int64_t i = FirstPiece(); i < pieces; i += PieceStride()) {
    const Piece piece = PieceOf(i, segments);
    const int64_t first = int64_t(piece.segment) * (64 * kValues * kUnits);
    int64_t at[kUnits];
    float sum[kUnits][kValues] = {};
#pragma unroll
    for (int u = 0; u < kUnits; ++u) at[u] = min(first + (u * 64 + lane) * kValues, int64_t(c.width) - kValues);
    for (int j0 = 0; j0 < c.top; j0 += kAtOnce) {
      v4i held[kAtOnce][kUnits][1];
      int place[kAtOnce];
      float weight[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        place[j] = j0 + j < c.top ? PlaceOf(c, piece.token, j0 + j) : -1;
        if (place[j] < 0) continue;
        weight[j] = WeightOf(c, piece.token, j0 + j);
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
          if (first + u * 64 * kValues < c.width) Load<kType, kValues>(c.place_side.data, place[j] * c.place_side.cs + at[u], held[j][u]);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (place[j] < 0) continue;
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
#pragma unroll
          for (int e = 0; e < kValues; ++e) sum[u][e] += weight[j] * Value<kType, kValues>(held[j][u], e);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
      if (first + u * 64 * kValues < c.width)
        Store<kDstType, kValues, kStreamed>(c.token_side.data, piece.token * c.token_side.cs + at[u], sum[u]);
  }
}

// ---- The same for narrow tokens ----
//
// A token of so few units that kLanes lanes have one each: 64 / kLanes tokens to a wave. (us, 100000 tokens of 128 values in bfloat16 with two
// places each, a wave to a token and these: to their places 24 and 10, added up 70 and 15, gradients 64 and 30; 12991 tokens of 151 values
// in half added up 9.9 and 5.5.)

template <int kBytes, int kLanes, bool kStreamed>
__global__ __launch_bounds__(256) void NarrowDispatchKernel(Call c) {
  const int64_t bytes = int64_t(c.width) * kBytes;
  const int first = (threadIdx.x & (kLanes - 1)) * 16;
  if (first >= bytes) return;
  const int64_t at = min(int64_t(first), bytes - 16);
  for (int64_t token = (int64_t(blockIdx.x) * 256 + threadIdx.x) / kLanes; token < c.tokens; token += int64_t(gridDim.x) * (256 / kLanes)) {
    const v4i held =
        *reinterpret_cast<const v4i_unaligned*>(static_cast<const char*>(c.token_side.data) + token * c.token_side.cs * kBytes + at);
    for (int j = 0; j < c.top; ++j) {
      const int place = PlaceOf(c, token, j);
      if (place >= 0)
        StoreGranule<kStreamed>(
            reinterpret_cast<v4i_unaligned*>(static_cast<char*>(c.place_side.data) + place * c.place_side.cs * kBytes + at), held);
    }
  }
}

template <int kType, int kDstType, int kLanes, bool kStreamed>
__global__ __launch_bounds__(256) void NarrowCombineKernel(Call c) {
  constexpr int kValues = 16 / Bytes(kType), kAtOnce = 4;
  const int first = (threadIdx.x & (kLanes - 1)) * kValues;
  if (first >= c.width) return;
  const int64_t at = min(first, c.width - kValues);
  for (int64_t token = (int64_t(blockIdx.x) * 256 + threadIdx.x) / kLanes; token < c.tokens; token += int64_t(gridDim.x) * (256 / kLanes)) {
    float sum[kValues] = {};
    for (int j0 = 0; j0 < c.top; j0 += kAtOnce) {
      v4i held[kAtOnce][1];
      int place[kAtOnce];
      float weight[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) place[j] = j0 + j < c.top ? PlaceOf(c, token, j0 + j) : -1;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (place[j] < 0) continue;
        weight[j] = WeightOf(c, token, j0 + j);
        Load<kType, kValues>(c.place_side.data, place[j] * c.place_side.cs + at, held[j]);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (place[j] < 0) continue;
#pragma unroll
        for (int e = 0; e < kValues; ++e) sum[e] += weight[j] * Value<kType, kValues>(held[j], e);
      }
    }
    Store<kDstType, kValues, kStreamed>(c.token_side.data, token * c.token_side.cs + at, sum);
  }
}

// ---- The gradients of that sum ----

// The lanes' values added up, in every lane, always in the same order: over 2, 4, 8 and 16 neighbours, then over the four rows of 16.
template <int kExchange>
__device__ __forceinline__ float Exchanged(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kExchange, 0xf, 0xf, true));
}
__device__ __forceinline__ float WaveSum(float v) {
  v += Exchanged<0xb1>(v);   // lanes 1 0 3 2
  v += Exchanged<0x4e>(v);   // lanes 2 3 0 1
  v += Exchanged<0x141>(v);  // eight lanes backwards
  v += Exchanged<0x140>(v);  // sixteen lanes backwards
  const int w = __float_as_int(v);
  const auto rows = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  v = __int_as_float(rows[0]) + __int_as_float(rows[1]);
  const int x = __float_as_int(v);
  const auto halves = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __int_as_float(halves[0]) + __int_as_float(halves[1]);
}

constexpr int kMostWaves = 8;

// `waves` waves to a token, whole tokens to a workgroup; the waves of a token take 64 * kUnits units in turn. kDots: choices at a time.
template <int kType, int kGradType, int kDots, int kUnits, bool kStreamed>
__global__ __launch_bounds__(64 * kMostWaves) void GradientsKernel(Call c, int waves) {
  constexpr int kValues = 16 / Bytes(kType), kUnit = 64 * kValues;
  __shared__ float dots[kMostWaves][kDots];
  const int lane = threadIdx.x & 63, my_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tokens_here = (blockDim.x >> 6) / waves, wave = my_wave % waves;
  const bool rows = c.grad_src.data, weights = c.grad_weights.data;
  for (int64_t token0 = int64_t(blockIdx.x) * tokens_here; token0 < c.tokens; token0 += int64_t(gridDim.x) * tokens_here) {
    const int64_t token = token0 + my_wave / waves;
    const bool there = token < c.tokens;  // (all waves go through the barriers)
    for (int j0 = 0; j0 < c.top; j0 += kDots) {
      int place[kDots];
      float weight[kDots], dot[kDots] = {};
#pragma unroll
      for (int j = 0; j < kDots; ++j) {
        place[j] = there && j0 + j < c.top ? PlaceOf(c, token, j0 + j) : -1;
        weight[j] = place[j] >= 0 && rows ? WeightOf(c, token, j0 + j) : 0.0f;
      }
      for (int64_t first = int64_t(wave) * (kUnit * kUnits); there && first < c.width; first += int64_t(waves) * (kUnit * kUnits)) {
        int64_t at[kUnits];
        v4i grad[kUnits][kValues * Bytes(kGradType) / 16], held[kDots][kUnits][1];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          at[u] = min(first + u * kUnit + lane * kValues, int64_t(c.width) - kValues);
          if (first + u * kUnit < c.width) Load<kGradType, kValues>(c.token_side.data, token * c.token_side.cs + at[u], grad[u]);
        }
        if (weights) {
#pragma unroll
          for (int j = 0; j < kDots; ++j)
#pragma unroll
            for (int u = 0; u < kUnits; ++u)
              if (place[j] >= 0 && first + u * kUnit < c.width)
                Load<kType, kValues>(c.place_side.data, place[j] * c.place_side.cs + at[u], held[j][u]);
        }
        if (rows) {
#pragma unroll
          for (int j = 0; j < kDots; ++j) {
            if (place[j] < 0) continue;
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
              if (first + u * kUnit >= c.width) continue;
              float v[kValues];
#pragma unroll
              for (int e = 0; e < kValues; ++e) v[e] = weight[j] * Value<kGradType, kValues>(grad[u], e);
              Store<kType, kValues, kStreamed>(c.grad_src.data, place[j] * c.grad_src.cs + at[u], v);
            }
          }
        }
        if (weights) {
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {
            if (first + u * kUnit >= c.width) continue;
            // (Values that the lane before has too.)
            const int again = static_cast<int>(min(first + u * kUnit + lane * kValues - at[u], int64_t(kValues)));
            float g[kValues];
#pragma unroll
            for (int e = 0; e < kValues; ++e) g[e] = Value<kGradType, kValues>(grad[u], e);
#pragma unroll
            for (int j = 0; j < kDots; ++j) {
              if (place[j] < 0) continue;
              if (first + (u + 1) * kUnit <= c.width) {  // (none)
#pragma unroll
                for (int e = 0; e < kValues; ++e) dot[j] += g[e] * Value<kType, kValues>(held[j][u], e);
              } else {
#pragma unroll
                for (int e = 0; e < kValues; ++e) {
                  const float product = g[e] * Value<kType, kValues>(held[j][u], e);
                  dot[j] += e >= again ? product : 0.0f;
                }
              }
            }
          }
        }
      }
      if (!weights) continue;
      float mine = 0;  // lane j's: choice j
#pragma unroll
      for (int j = 0; j < kDots; ++j) {
        if (j0 + j >= c.top) break;
        const float sum = WaveSum(dot[j]);
        mine = lane == j ? sum : mine;
      }
      if (waves > 1) {
        if (lane < kDots) dots[my_wave][lane] = mine;
        __syncthreads();
        mine = 0;
        if (wave == 0 && lane < kDots)
          for (int w = 0; w < waves; ++w) mine += dots[my_wave + w][lane];
        __syncthreads();
      }
      if (there && wave == 0 && lane < kDots && j0 + lane < c.top)
        StoreFloat(c.grad_weights.data, c.grad_weights.type, (j0 + lane) * c.grad_weights.rs + token * c.grad_weights.cs, mine);
    }
  }
}

// Narrow tokens, kLanes lanes to each (as above).
template <int kType, int kGradType, int kLanes, bool kStreamed>
__global__ __launch_bounds__(256) void NarrowGradientsKernel(Call c) {
  constexpr int kValues = 16 / Bytes(kType), kAtOnce = 4;
  const int mine = threadIdx.x & (kLanes - 1), first = mine * kValues;
  const bool active = first < c.width;  // (all lanes go through the sums)
  const int64_t at = min(first, c.width - kValues);
  const int again = static_cast<int>(min(int64_t(first) - at, int64_t(kValues)));  // values that the lane before has too
  const bool rows = c.grad_src.data, weights = c.grad_weights.data;
  const int64_t tokens_here = 256 / kLanes, stride = int64_t(gridDim.x) * tokens_here;
  for (int64_t token0 = int64_t(blockIdx.x) * tokens_here; token0 < c.tokens; token0 += stride) {
    const int64_t token = token0 + threadIdx.x / kLanes;
    const bool there = active && token < c.tokens;
    v4i raw[kValues * Bytes(kGradType) / 16];
    float grad[kValues] = {};
    if (there) {
      Load<kGradType, kValues>(c.token_side.data, token * c.token_side.cs + at, raw);
#pragma unroll
      for (int e = 0; e < kValues; ++e) grad[e] = Value<kGradType, kValues>(raw, e);
    }
    for (int j0 = 0; j0 < c.top; j0 += kAtOnce) {
      int place[kAtOnce];
      v4i held[kAtOnce][1];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) place[j] = there && j0 + j < c.top ? PlaceOf(c, token, j0 + j) : -1;
      if (weights) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
          if (place[j] >= 0) Load<kType, kValues>(c.place_side.data, place[j] * c.place_side.cs + at, held[j]);
      }
      if (rows) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          if (place[j] < 0) continue;
          const float weight = WeightOf(c, token, j0 + j);
          float v[kValues];
#pragma unroll
          for (int e = 0; e < kValues; ++e) v[e] = weight * grad[e];
          Store<kType, kValues, kStreamed>(c.grad_src.data, place[j] * c.grad_src.cs + at, v);
        }
      }
      if (weights) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          if (j0 + j >= c.top) break;
          float dot = 0;
          if (place[j] >= 0) {
#pragma unroll
            for (int e = 0; e < kValues; ++e) {
              const float product = grad[e] * Value<kType, kValues>(held[j], e);
              dot += e >= again ? product : 0.0f;
            }
          }
#pragma unroll
          for (int d = 1; d < kLanes; d *= 2) dot += __shfl_xor(dot, d);
          if (mine == 0 && there)
            StoreFloat(c.grad_weights.data, c.grad_weights.type, (j0 + j) * c.grad_weights.rs + token * c.grad_weights.cs, dot);
        }
      }
    }
  }
}

// ---- One value to a lane ----

constexpr unsigned kMostBlocks = 1u << 20;
unsigned BlocksFor(int64_t work, int threads) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((work + threads - 1) / threads, kMostBlocks)));
}
// A value of a token and the token; the former is the fast one where values lie side by side.
__device__ __forceinline__ void TokenAndValue(const Call& c, bool by_values, int64_t i, int* token, int* value) {
  const int fast = by_values ? c.width : c.tokens;
  const int slow = static_cast<int>(i / fast), rest = static_cast<int>(i - int64_t(slow) * fast);
  *token = by_values ? slow : rest;
  *value = by_values ? rest : slow;
}

__global__ __launch_bounds__(256) void GenericDispatchKernel(Call c) {
  const int64_t all = int64_t(c.tokens) * c.width;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(gridDim.x) * 256) {
    int token, h;
    TokenAndValue(c, c.token_side.rs == 1, i, &token, &h);
    const int64_t from = h * c.token_side.rs + token * c.token_side.cs;
    for (int j = 0; j < c.top; ++j) {
      const int place = PlaceOf(c, token, j);
      if (place < 0) continue;
      const int64_t to = h * c.place_side.rs + place * c.place_side.cs;
      if (c.token_side.type == RUYAMD_DTYPE_F32)
        static_cast<uint32_t*>(c.place_side.data)[to] = static_cast<const uint32_t*>(c.token_side.data)[from];
      else
        static_cast<uint16_t*>(c.place_side.data)[to] = static_cast<const uint16_t*>(c.token_side.data)[from];
    }
  }
}

__global__ __launch_bounds__(256) void GenericCombineKernel(Call c) {
  const int64_t all = int64_t(c.tokens) * c.width;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(gridDim.x) * 256) {
    int token, h;
    TokenAndValue(c, c.token_side.rs == 1, i, &token, &h);
    float sum = 0;
    for (int j = 0; j < c.top; ++j) {
      const int place = PlaceOf(c, token, j);
      if (place >= 0)
        sum += WeightOf(c, token, j) * LoadFloat(c.place_side.data, c.place_side.type, h * c.place_side.rs + place * c.place_side.cs);
    }
    StoreFloat(c.token_side.data, c.token_side.type, h * c.token_side.rs + token * c.token_side.cs, sum);
  }
}

__global__ __launch_bounds__(256) void GenericRowGradientsKernel(Call c) {
  const int64_t all = int64_t(c.tokens) * c.width;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(gridDim.x) * 256) {
    int token, h;
    TokenAndValue(c, c.token_side.rs == 1, i, &token, &h);
    const float grad = LoadFloat(c.token_side.data, c.token_side.type, h * c.token_side.rs + token * c.token_side.cs);
    for (int j = 0; j < c.top; ++j) {
      const int place = PlaceOf(c, token, j);
      if (place >= 0)
        StoreFloat(c.grad_src.data, c.grad_src.type, h * c.grad_src.rs + place * c.grad_src.cs, WeightOf(c, token, j) * grad);
    }
  }
}

// A wave to a choice.
__global__ __launch_bounds__(256) void GenericWeightGradientsKernel(Call c) {
  const int lane = threadIdx.x & 63;
  const int64_t choices = int64_t(c.tokens) * c.top;
  for (int64_t i = FirstPiece(); i < choices; i += PieceStride()) {
    const Piece choice = PieceOf(i, c.top);
    const int place = PlaceOf(c, choice.token, choice.segment);
    float sum = 0;
    if (place >= 0)
      for (int64_t h = lane; h < c.width; h += 64)
        sum += LoadFloat(c.token_side.data, c.token_side.type, h * c.token_side.rs + choice.token * c.token_side.cs) *
               LoadFloat(c.place_side.data, c.place_side.type, h * c.place_side.rs + place * c.place_side.cs);
    sum = WaveSum(sum);
    if (lane == 0)
      StoreFloat(c.grad_weights.data, c.grad_weights.type, choice.segment * c.grad_weights.rs + choice.token * c.grad_weights.cs, sum);
  }
}

// Whether a view's values of a token lie side by side (one value alone does).
bool SideBySide(const Call& c, const View& v) { return !v.data || v.rs == 1 || c.width == 1; }

// Segments of 64 * units units of 16 bytes, and how many units: no more than a row has (100000 tokens of 512 values in bfloat16 added up with
// four units 72.7 us, with one 49.7), and as many as leave every CU some waves. f(units as a
// constant, segments, blocks).
template <class F>
void WithUnits(const Call& c, int type, int compute_units, F&& f) {
  const int64_t unit = 64 * (16 / Bytes(type));
  const auto segments = [&](int units) { return (c.width + unit * units - 1) / (unit * units); };
  const auto blocks = [&](int64_t s) { return BlocksFor(c.tokens * s, 4); };
  const int64_t enough = int64_t(16) * compute_units;
  if (c.width > 2 * unit && c.tokens * segments(4) >= enough) return f(std::integral_constant<int, 4>(), int(segments(4)), blocks(segments(4)));
  if (c.width > unit && c.tokens * segments(2) >= enough) return f(std::integral_constant<int, 2>(), int(segments(2)), blocks(segments(2)));
  f(std::integral_constant<int, 1>(), int(segments(1)), blocks(segments(1)));
}

// Bytes written from which on they go past the caches: 32 MiB, which is what all L2s hold. (Rows that are whole lines; us, tokens of 4096 values in bfloat16 and two
// places each, 17, 34, 67 and 134 MB dispatched: 6.7 10.1 24.3 41.8, past them 5.5 9.0 16.7 32.7; combined, 8, 17, 34 and 67 MB: 6.4 9.6 22.8
// 41.5, past them 5.9 9.6 17.3 37.9; combined and dispatched again, 2048 tokens 18.8 and 21.0, 4096 44.7 and 40.0.)
constexpr int64_t kStreamFrom = int64_t(1) << 25;
template <class F>
void WithStores(int64_t bytes, F&& f) {
  if (bytes >= kStreamFrom) return f(std::true_type());
  f(std::false_type());
}

// Lanes to a narrow token: f(lanes as a constant), or false for one that is not narrow.
template <class F>
bool WithLanes(const Call& c, int type, F&& f) {
  const int64_t units = (int64_t(c.width) * Bytes(type) + 15) / 16;
  if (units > 32) return false;
  if (units > 16)
    f(std::integral_constant<int, 32>());
  else if (units > 8)
    f(std::integral_constant<int, 16>());
  else
    f(std::integral_constant<int, 8>());
  return true;
}

// f(type of the rows, other type): the other is the rows' or fp32.
template <class F>
void WithTypes(int type, int other, F&& f) {
  using BF16 = std::integral_constant<int, RUYAMD_DTYPE_BF16>;
  using F16 = std::integral_constant<int, RUYAMD_DTYPE_F16>;
  using F32 = std::integral_constant<int, RUYAMD_DTYPE_F32>;
  if (type == RUYAMD_DTYPE_F32) return f(F32(), F32());
  if (type == RUYAMD_DTYPE_BF16) return other == type ? f(BF16(), BF16()) : f(BF16(), F32());
  return other == type ? f(F16(), F16()) : f(F16(), F32());
}

}  // namespace

bool LaunchDispatch(hipStream_t stream, const Call& c, int compute_units, hipError_t* status) {
  const int type = c.token_side.type;
  if (c.width < 16 / Bytes(type) || !SideBySide(c, c.token_side) || !SideBySide(c, c.place_side)) return false;
  const bool narrow = WithLanes(c, type, [&](auto lanes) {
    constexpr int kLanes = decltype(lanes)::value;
    WithStores(int64_t(c.tokens) * c.top * c.width * Bytes(type), [&](auto streamed) {
      constexpr bool kStreamed = decltype(streamed)::value;
      const dim3 grid(BlocksFor(int64_t(c.tokens) * kLanes, 256));
      if (type == RUYAMD_DTYPE_F32)
        hipLaunchKernelGGL((NarrowDispatchKernel<4, kLanes, kStreamed>), grid, dim3(256), 0, stream, c);
      else
        hipLaunchKernelGGL((NarrowDispatchKernel<2, kLanes, kStreamed>), grid, dim3(256), 0, stream, c);
    });
  });
  if (!narrow) WithUnits(c, type, compute_units, [&](auto units, int segments, unsigned blocks) {
    constexpr int kUnits = decltype(units)::value;
    WithStores(int64_t(c.tokens) * c.top * c.width * Bytes(type), [&](auto streamed) {
      constexpr bool kStreamed = decltype(streamed)::value;
      if (type == RUYAMD_DTYPE_F32)
        hipLaunchKernelGGL((DispatchKernel<4, kUnits, kStreamed>), dim3(blocks), dim3(256), 0, stream, c, segments);
      else
        hipLaunchKernelGGL((DispatchKernel<2, kUnits, kStreamed>), dim3(blocks), dim3(256), 0, stream, c, segments);
    });
  });
  *status = hipGetLastError();
  return true;
}

bool LaunchCombine(hipStream_t stream, const Call& c, int compute_units, hipError_t* status) {
  const int type = c.place_side.type;
  if (c.width < 16 / Bytes(type) || !SideBySide(c, c.token_side) || !SideBySide(c, c.place_side)) return false;
  const bool narrow = WithLanes(c, type, [&](auto lanes) {
    WithTypes(type, c.token_side.type, [&](auto t, auto dst) {
      constexpr int kType = decltype(t)::value, kDst = decltype(dst)::value, kLanes = decltype(lanes)::value;
      WithStores(int64_t(c.tokens) * c.width * Bytes(kDst), [&](auto streamed) {
        hipLaunchKernelGGL((NarrowCombineKernel<kType, kDst, kLanes, decltype(streamed)::value>),
                           dim3(BlocksFor(int64_t(c.tokens) * kLanes, 256)), dim3(256), 0, stream, c);
      });
    });
  });
  if (!narrow) WithUnits(c, type, compute_units, [&](auto units, int segments, unsigned blocks) {
    WithTypes(type, c.token_side.type, [&](auto t, auto dst) {
      constexpr int kType = decltype(t)::value, kDst = decltype(dst)::value, kUnits = decltype(units)::value;
      WithStores(int64_t(c.tokens) * c.width * Bytes(kDst), [&](auto streamed) {
        hipLaunchKernelGGL((CombineKernel<kType, kDst, kUnits, decltype(streamed)::value>), dim3(blocks), dim3(256), 0, stream, c, segments);
      });
    });
  });
  *status = hipGetLastError();
  return true;
}

bool LaunchGradients(hipStream_t stream, const Call& c, int compute_units, hipError_t* status) {
  const int type = c.place_side.type;
  if (c.width < 16 / Bytes(type) || !SideBySide(c, c.token_side) || !SideBySide(c, c.place_side) || !SideBySide(c, c.grad_src))
    return false;
  const bool narrow = WithLanes(c, type, [&](auto lanes) {
    WithTypes(type, c.token_side.type, [&](auto t, auto grad) {
      constexpr int kType = decltype(t)::value, kGrad = decltype(grad)::value, kLanes = decltype(lanes)::value;
      WithStores(c.grad_src.data ? int64_t(c.tokens) * c.top * c.width * Bytes(kType) : 0, [&](auto streamed) {
        hipLaunchKernelGGL((NarrowGradientsKernel<kType, kGrad, kLanes, decltype(streamed)::value>),
                           dim3(BlocksFor(int64_t(c.tokens) * kLanes, 256)), dim3(256), 0, stream, c);
      });
    });
  });
  if (narrow) {
    *status = hipGetLastError();
    return true;
  }
  // Waves to a token: as few as leave every CU 16, each with a unit at least.
  const int64_t units = (c.width + 64 * (16 / Bytes(type)) - 1) / (64 * (16 / Bytes(type)));
  int waves = 1;
  while (waves < kMostWaves && waves < units && int64_t(c.tokens) * waves < int64_t(16) * compute_units) waves *= 2;
  const int block = std::max(waves, 4);
  const dim3 grid(BlocksFor(int64_t(c.tokens) * waves, block)), threads(64 * block);
  WithTypes(type, c.token_side.type, [&](auto t, auto grad) {
    constexpr int kType = decltype(t)::value, kGrad = decltype(grad)::value;
    WithStores(c.grad_src.data ? int64_t(c.tokens) * c.top * c.width * Bytes(kType) : 0, [&](auto streamed) {
      constexpr bool kStreamed = decltype(streamed)::value;
      if (c.top <= 2)
        hipLaunchKernelGGL((GradientsKernel<kType, kGrad, 2, 2, kStreamed>), grid, threads, 0, stream, c, waves);
      else if (c.top <= 4)
        hipLaunchKernelGGL((GradientsKernel<kType, kGrad, 4, 2, kStreamed>), grid, threads, 0, stream, c, waves);
      else
        hipLaunchKernelGGL((GradientsKernel<kType, kGrad, 8, 1, kStreamed>), grid, threads, 0, stream, c, waves);
    });
  });
  *status = hipGetLastError();
  return true;
}

hipError_t LaunchGenericDispatch(hipStream_t stream, const Call& c) {
  hipLaunchKernelGGL(GenericDispatchKernel, dim3(BlocksFor(int64_t(c.tokens) * c.width, 256)), dim3(256), 0, stream, c);
  return hipGetLastError();
}
hipError_t LaunchGenericCombine(hipStream_t stream, const Call& c) {
  hipLaunchKernelGGL(GenericCombineKernel, dim3(BlocksFor(int64_t(c.tokens) * c.width, 256)), dim3(256), 0, stream, c);
  return hipGetLastError();
}
hipError_t LaunchGenericGradients(hipStream_t stream, const Call& c) {
  if (c.grad_src.data && c.width)
    hipLaunchKernelGGL(GenericRowGradientsKernel, dim3(BlocksFor(int64_t(c.tokens) * c.width, 256)), dim3(256), 0, stream, c);
  if (c.grad_weights.data)
    hipLaunchKernelGGL(GenericWeightGradientsKernel, dim3(BlocksFor(int64_t(c.tokens) * c.top, 4)), dim3(256), 0, stream, c);
  return hipGetLastError();
}

}  // namespace routing
}  // namespace ruyamd
