// Device helpers shared by the serving attention kernels.
#pragma once
#include "../../include/iris_b200.h"
#include "detnum.cuh"
#include "serve.cuh"

namespace iris {

constexpr uint32_t kServeMaxDim = 256;  // widest head

// The score of a wrapped Q32.32 dot product: scaled (mistral.rs:130-145), or
// requantized as it is where scale is 0 (gemma-dense).
__device__ __forceinline__ int32_t serve_score(int64_t sum, uint32_t scale) {
  return scale ? scaled_score_finish(sum, scale) : requantize(sum);
}

__device__ __forceinline__ unsigned long long node_bits(uint32_t nodes) {
  return nodes >= 64 ? ~0ull : (1ull << nodes) - 1;
}

// A request's cached tokens, held inside what its table and `longest` cover.
__device__ __forceinline__ uint32_t tree_held(const IrisTreeAttention& a, uint32_t r) {
  return min((uint32_t)max(a.held[r], 0), a.longest);
}

// Whether a node of visible nodes `mask` at `position` sees the key at index
// `at` of its request: the cached tokens come first, then the nodes. A window
// hides keys whose position is `window` or more below (positions: the nodes').
__device__ __forceinline__ bool tree_sees(uint32_t at, uint32_t held, unsigned long long mask, uint32_t window,
                                          uint32_t position, const int32_t* positions) {
  if (at < held) return !window || at + window > position;
  const uint32_t node = at - held;
  return node < kTreeNodes && (mask >> node & 1) && (!window || (uint32_t)positions[node] + window > position);
}

}  // namespace iris
