// Drafted trees over the paged cache: what the launches on the matrix
// instructions (tree_mma.cu) and on the tcgen05 tensor cores (tree_tc.cu) share.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/iris_b200.h"
#include "layers.cuh"
#include "serve_attn.cuh"

namespace iris {

struct TreeScratch {
  int32_t* scores;     // [rows * heads][pitch], then terms
  int32_t* chunk_max;  // [rows * heads][chunks]
  uint64_t* seg_sum;   // [rows * heads][segs]
  uint32_t* seg_first; // [rows * heads][segs]
  int64_t* acc;        // [rows * heads][d]
  int32_t* wsum;       // [rows * heads]
  uint32_t* done;      // [requests][kv_heads][groups]: finished blocks of the third launch
  uint32_t pitch, chunk, chunks, segs;
  uint32_t vchunk, vchunks, groups;  // keys and row groups of the third launch's blocks
  // on the tensor cores: flags[0] a query or key, flags[1] a value past 24
  // bits (the launches of tree_mma.cu behind then do the work), and totals of
  // their own; NULL otherwise
  uint32_t* flags;
  int64_t* tc_acc;
  int32_t* tc_wsum;
  uint32_t* tc_done;  // [requests][kv_heads][tc_groups]
  uint32_t tc_groups, tc_rows, tc_vchunk, tc_vchunks;
};

constexpr uint32_t kTreeSegment = 1024;  // keys a warp takes in the second launch
constexpr uint32_t kTreeTcRows = 256;    // query rows of a tensor-core scores block

// One request's part of the call: its keys from `base` on (a multiple of 64; a
// window hides all below from every node). Made by whole warps.
struct TreeRequest {
  uint32_t begin, nodes, held, keys, group, base, count;
  uint32_t inverse;  // of the group, rounded up: floor(f inverse / 2^32) is f / group for f and group up to 2^16
  __device__ TreeRequest(const IrisTreeAttention& a, uint32_t r) {
    begin = clamp_offset(a.offsets[r], a.rows);
    const uint32_t end = clamp_offset(a.offsets[r + 1], a.rows);
    nodes = end > begin ? min(end - begin, a.nodes) : 0;
    held = tree_held(a, r);
    keys = min(held + nodes, a.longest);
    group = a.heads / a.kv_heads;
    inverse = 0xFFFFFFFFu / group + 1;
    base = 0;
    if (a.window) {
      uint32_t low = held;
      for (uint32_t i = threadIdx.x & 31; i < nodes; i += 32)
        low = min(low, window_start((uint32_t)a.positions[begin + i], a.window));
      base = min(__reduce_min_sync(0xffffffffu, low), keys) / 64 * 64;
    }
    count = keys - base;
  }
  // The node of a K/V head's row f (node * group + head), and its query head.
  __device__ uint32_t node_of(uint32_t f) const { return group == 1 ? f : __umulhi(f, inverse); }
  __device__ uint32_t head_of(uint32_t f, uint32_t g) const { return g * group + f - node_of(f) * group; }
};

// The pool row that is read for keys that are not there (past the request's end or
// off its table; they are masked, and their weights 0): the row of the request's
// last key, so that only rows the call names choose its arithmetic.
__device__ __forceinline__ uint32_t stand_in_row(const IrisTreeAttention& a, const TreeRequest& q, const int32_t* table) {
  return (uint32_t)max(page_row(table, a.width, a.page_size, a.pages, q.keys - 1), (int64_t)0);
}

// head_dim up to 128 and trees of enough rows.
bool tree_tc_usable(const IrisTreeAttention& a);
// The scores and the value sums; flags are cleared before, terms run between.
cudaError_t launch_tree_tc_scores(const IrisTreeAttention& a, const TreeScratch& sc, cudaStream_t stream);
cudaError_t launch_tree_tc_values(const IrisTreeAttention& a, const TreeScratch& sc, cudaStream_t stream);

}  // namespace iris
