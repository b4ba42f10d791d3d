// Attention of drafted trees over the paged cache on the matrix instructions.
//
// The work is split over the keys, so that a few rows over a long context use
// every multiprocessor, and joined exactly: maxima, sums of terms and value
// sums are integers, whose order of addition does not matter. Three launches:
//   1. scores: a block takes a chunk of one request's keys for one K/V head
//      and all the query rows that share it, writes the scores and each row's
//      maximum over the chunk;
//   2. terms: a warp takes a segment of one row: the row's maximum over the
//      chunks, the exponential of every score in place, their sum and the
//      first maximum's place;
//   3. values: a block takes a chunk of keys again: the row's sum over the
//      segments, weights, value sums added to the row's 64-bit totals; the
//      last block of a request and K/V head adds the first maximum's weight
//      (1.0 less the others) and writes the outputs.
// K and V cross HBM once each; the scores (4 bytes a row and key, a fraction of
// the keys' 512) stay in L2 between the launches.
#include <algorithm>

#include "../../include/iris_b200.h"
#include "common.cuh"
#include "layers.cuh"
#include "serve_attn.cuh"
#include "serve_mma.cuh"
#include "tree_mma.cuh"

namespace iris {

namespace {

constexpr uint32_t kTreeThreads = 256, kTreeWarps = kTreeThreads / 32;
constexpr uint32_t kTreeTile = 32;     // query rows a block works on at a time
constexpr uint32_t kTreeSegment = 1024;  // keys a warp takes in the second launch

struct TreeScratch {
  int32_t* scores;     // [rows * heads][pitch], then terms
  int32_t* chunk_max;  // [rows * heads][chunks]
  uint64_t* seg_sum;   // [rows * heads][segs]
  uint32_t* seg_first; // [rows * heads][segs]
  int64_t* acc;        // [rows * heads][d]
  int32_t* wsum;       // [rows * heads]
  uint32_t* done;      // [requests * kv_heads]
  uint32_t pitch, chunk, chunks, segs;
};

// One request's part of the call: its keys from `base` on (a multiple of 64; a
// window hides all below from every node). Made by whole warps.
struct TreeRequest {
  uint32_t begin, nodes, held, keys, group, base, count;
  __device__ TreeRequest(const IrisTreeAttention& a, uint32_t r) {
    begin = clamp_offset(a.offsets[r], a.rows);
    const uint32_t end = clamp_offset(a.offsets[r + 1], a.rows);
    nodes = end > begin ? min(end - begin, a.nodes) : 0;
    held = tree_held(a, r);
    keys = min(held + nodes, a.longest);
    group = a.heads / a.kv_heads;
    base = 0;
    if (a.window) {
      uint32_t low = held;
      for (uint32_t i = threadIdx.x & 31; i < nodes; i += 32)
        low = min(low, window_start((uint32_t)a.positions[begin + i], a.window));
      base = min(__reduce_min_sync(0xffffffffu, low), keys) / 64 * 64;
    }
    count = keys - base;
  }
};

__device__ __forceinline__ bool is_visible(const IrisTreeAttention& a, const TreeRequest& q, uint32_t node,
                                           uint32_t key) {
  const uint32_t row = q.begin + node;
  return tree_sees(key, q.held, (unsigned long long)a.masks[row] & node_bits(q.nodes), a.window,
                   a.positions ? (uint32_t)a.positions[row] : 0, a.positions + q.begin);
}

__global__ void __launch_bounds__(kTreeThreads, 2) tree_scores_kernel(IrisTreeAttention a, TreeScratch sc) {
  extern __shared__ __align__(16) uint8_t tree_sm[];
  uint2* frag = (uint2*)tree_sm;  // [tile / 8][steps][4][32]
  __shared__ int32_t row_max[kTreeTile];
  __shared__ uint32_t q_wide;
  const uint32_t chunk = blockIdx.x, g = blockIdx.y, r = blockIdx.z;
  const TreeRequest q(a, r);
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, steps = a.head_dim / 32;
  const uint32_t rows = q.nodes * q.group, key0 = q.base + chunk * sc.chunk;
  if (chunk == 0) {  // the totals of this request and head start at zero
    for (uint32_t i = tid; i < rows * a.head_dim; i += kTreeThreads) {
      const uint32_t f = i / a.head_dim, x = i % a.head_dim;
      const size_t id = (size_t)(q.begin + f / q.group) * a.heads + g * q.group + f % q.group;
      sc.acc[id * a.head_dim + x] = 0;
      if (x == 0) sc.wsum[id] = 0;
    }
    if (tid == 0) sc.done[r * a.kv_heads + g] = 0;
  }
  if (key0 >= q.keys) return;
  const uint32_t key1 = min(key0 + sc.chunk, q.base + (q.count + 15) / 16 * 16);
  const int32_t* table = a.table + (size_t)r * a.width;
  const size_t kvd = (size_t)a.kv_heads * a.head_dim;
  const QueryTile tile{frag, steps};
  for (uint32_t f0 = 0; f0 < rows; f0 += kTreeTile) {
    if (f0) __syncthreads();
    if (tid < kTreeTile) row_max[tid] = INT32_MIN;
    if (tid == 0) q_wide = 0;
    __syncthreads();
    for (uint32_t u = warp; u < kTreeTile / 8 * steps; u += kTreeWarps) {
      const uint32_t nt = u / steps, f = f0 + 8 * nt + (lane >> 2);
      const int32_t* src = nullptr;
      if (f < rows)
        src = a.q + (size_t)(q.begin + f / q.group) * a.q_stride + (g * q.group + f % q.group) * a.head_dim;
      if (put_query_fragment(frag, steps, nt, u % steps, lane, src)) q_wide = 1;
    }
    __syncthreads();
    const bool wide = q_wide != 0;
    for (uint32_t t0 = key0 + 16 * warp; t0 < key1; t0 += 16 * kTreeWarps) {
      const uint32_t ka = t0 + (lane >> 2), kb = ka + 8;
      const int64_t ra = ka < q.keys ? page_row(table, a.width, a.page_size, a.pages, ka) : -1;
      const int64_t rb = kb < q.keys ? page_row(table, a.width, a.page_size, a.pages, kb) : -1;
      const int32_t* pa = ra >= 0 ? a.k_pages + (size_t)ra * kvd + g * a.head_dim : nullptr;
      const int32_t* pb = rb >= 0 ? a.k_pages + (size_t)rb * kvd + g * a.head_dim : nullptr;
      // keys that every row sees need no look at the masks
      const bool open = t0 + 16 <= q.held && !a.window && __all_sync(0xffffffffu, ra >= 0 && rb >= 0);
      int32_t best[2] = {INT32_MIN, INT32_MIN};
      uint32_t done = 0;
      key_scores<kTreeTile / 8>(pa, pb, tile, wide, 0, lane, a.scale_q32, [&](uint32_t n, uint32_t e, int32_t s) {
        const uint32_t f = f0 + 8 * n + 2 * (lane & 3) + (e & 1), key = e >> 1 ? kb : ka;
        if (f < rows) {
          if (!open && !((e >> 1 ? rb : ra) >= 0 && is_visible(a, q, f / q.group, key))) s = INT32_MIN;
          const size_t id = (size_t)(q.begin + f / q.group) * a.heads + g * q.group + f % q.group;
          sc.scores[id * sc.pitch + (key - q.base)] = s;
          best[e & 1] = max(best[e & 1], s);
        }
        if (++done % 4 == 0) {  // the four elements of these eight rows
          int32_t x = best[0], y = best[1];
#pragma unroll
          for (uint32_t o = 4; o <= 16; o <<= 1) {
            x = max(x, __shfl_xor_sync(0xffffffffu, x, o));
            y = max(y, __shfl_xor_sync(0xffffffffu, y, o));
          }
          if (lane < 4) {
            atomicMax(&row_max[8 * n + 2 * lane], x);
            atomicMax(&row_max[8 * n + 2 * lane + 1], y);
          }
          best[0] = best[1] = INT32_MIN;
        }
      });
    }
    __syncthreads();
    if (tid < kTreeTile && f0 + tid < rows) {
      const uint32_t f = f0 + tid;
      const size_t id = (size_t)(q.begin + f / q.group) * a.heads + g * q.group + f % q.group;
      sc.chunk_max[id * sc.chunks + chunk] = row_max[tid];
    }
  }
}

// Hidden keys carry the lowest score. Where the row's maximum is within 16.0 of
// it (every score saturated), that mark does not tell and the masks are asked
// again; elsewhere a key at the lowest score has term 0, seen or not.
__global__ void __launch_bounds__(kTreeThreads) tree_terms_kernel(IrisTreeAttention a, TreeScratch sc) {
  const uint32_t r = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t row = blockIdx.x * kTreeWarps + warp;  // node * heads + head
  const uint32_t seg = blockIdx.y;
  __shared__ uint32_t lists[kTreeWarps][kTermList];
  pdl_wait();
  pdl_trigger();
  const TreeRequest q(a, r);
  if (row >= q.nodes * a.heads || seg * kTreeSegment >= q.count) return;
  const uint32_t node = row / a.heads;
  const size_t id = (size_t)q.begin * a.heads + row;
  const uint32_t chunks = (q.count + sc.chunk - 1) / sc.chunk;
  int32_t top = INT32_MIN;
  for (uint32_t c = lane; c < chunks; c += 32) top = max(top, sc.chunk_max[id * sc.chunks + c]);
  top = __reduce_max_sync(0xffffffffu, top);
  const bool ask = top < INT32_MIN + (1 << 20);
  const uint32_t last = (q.count + 15) / 16 * 16;  // scores are written up to here
  const uint32_t s0 = seg * kTreeSegment, count = min(kTreeSegment, last - s0);
  const uint32_t stored = min(kTreeSegment, (q.count + 31) / 32 * 32 - s0);
  int32_t* s = sc.scores + id * sc.pitch + s0;
  uint64_t sum = 0;
  uint32_t first = UINT32_MAX;
  if (!ask) {
    int4 x[2];
    row_load(x, s, 128, 0, count, lane);
    const RowTerms t = row_terms(s, 128, count, stored, top, lists[warp], lane, x, nullptr);
    sum = t.sum;
    if (t.first != UINT32_MAX) first = s0 + t.first;
  } else {
    for (uint32_t t = lane; t < stored; t += 32) {
      const uint32_t key = q.base + s0 + t;
      const bool seen = key < q.keys && page_row(a.table + (size_t)r * a.width, a.width, a.page_size, a.pages, key) >= 0 &&
                        is_visible(a, q, node, key);
      const uint32_t e = seen ? term_of(__ldcg(s + t), top) : 0;
      if (e == kTermTop) first = min(first, s0 + t);
      sum += kept_term(e);
      __stcg((uint32_t*)s + t, e);
    }
  }
  sum = (uint64_t)warp_sum_i64((int64_t)sum);
  first = __reduce_min_sync(0xffffffffu, first);
  if (lane == 0) {
    sc.seg_sum[id * sc.segs + seg] = sum;
    sc.seg_first[id * sc.segs + seg] = first;
  }
}

template <uint32_t P>
__device__ __forceinline__ uint32_t tree_value_tile(const IrisTreeAttention& a, const TreeScratch& sc,
                                                    const TreeRequest& q, const uint2* w, const int64_t* row_s,
                                                    uint32_t steps, uint32_t g, uint32_t f0, uint32_t dt,
                                                    uint32_t step0, uint32_t step_by, uint32_t lane) {
  constexpr uint32_t NT = kTreeTile / 8;
  int32_t acc[NT][P + 1][4] = {};
  const int32_t* v = a.v_pages + g * a.head_dim + 16 * dt + 2 * (lane >> 2);
  const size_t kvd = (size_t)a.kv_heads * a.head_dim;
  uint32_t wide = 0;
  for (uint32_t st = step0; st < steps; st += step_by) {
    int2 x[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const int64_t row = row_s[st * 32 + (i >> 2) * 16 + 4 * (lane & 3) + (i & 3)];
      x[i] = row >= 0 ? *(const int2*)(v + (size_t)row * kvd) : make_int2(0, 0);
    }
    wide |= value_products<P, NT>(x, w + st * (NT * 64), lane, acc);
  }
  if (P == 3 && __any_sync(0xffffffffu, wide != 0)) return 1;
  const uint32_t rows = q.nodes * q.group;
#pragma unroll
  for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      const uint32_t f = f0 + 8 * n + 2 * (lane & 3) + (e & 1);
      if (f < rows) {
        int32_t d[P + 1];
#pragma unroll
        for (uint32_t j = 0; j < P + 1; ++j) d[j] = acc[n][j][e];
        const size_t id = (size_t)(q.begin + f / q.group) * a.heads + g * q.group + f % q.group;
        atomicAdd((unsigned long long*)(sc.acc + id * a.head_dim + 16 * dt + 2 * (lane >> 2) + (e >> 1)),
                  (unsigned long long)diagonal_sum(d));
      }
    }
  return 0;
}

__global__ void __launch_bounds__(kTreeThreads, 2) tree_values_kernel(IrisTreeAttention a, TreeScratch sc) {
  constexpr uint32_t NT = kTreeTile / 8;
  extern __shared__ __align__(16) uint8_t tree_sm[];
  uint2* w = (uint2*)tree_sm;                                   // [chunk / 32][NT][2][32]
  int64_t* row_s = (int64_t*)(w + (size_t)sc.chunk / 32 * NT * 64);  // [chunk]
  __shared__ uint64_t sum_s[kTreeTile];
  __shared__ uint32_t recip_s[kTreeTile], first_s[kTreeTile], last_s;
  const uint32_t chunk = blockIdx.x, g = blockIdx.y, r = blockIdx.z;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const TreeRequest q(a, r);
  const uint32_t rows = q.nodes * q.group, key0 = q.base + chunk * sc.chunk, s0 = chunk * sc.chunk;
  const uint32_t chunks = (q.count + sc.chunk - 1) / sc.chunk, segs = (q.count + kTreeSegment - 1) / kTreeSegment;
  if (!rows || key0 >= q.keys) return;
  const uint32_t count = min(sc.chunk, (q.keys - key0 + 31) / 32 * 32), steps = count / 32;
  for (uint32_t i = tid; i < count; i += kTreeThreads)
    row_s[i] = key0 + i < q.keys ? page_row(a.table + (size_t)r * a.width, a.width, a.page_size, a.pages, key0 + i) : -1;
  pdl_wait();
  for (uint32_t f0 = 0; f0 < rows; f0 += kTreeTile) {
    __syncthreads();
    for (uint32_t i = warp; i < kTreeTile; i += kTreeWarps) {
      const uint32_t f = f0 + i;
      uint64_t sum = 0;
      uint32_t first = UINT32_MAX;
      if (f < rows) {
        const size_t id = (size_t)(q.begin + f / q.group) * a.heads + g * q.group + f % q.group;
        for (uint32_t s = lane; s < segs; s += 32) {
          sum += sc.seg_sum[id * sc.segs + s];
          first = min(first, sc.seg_first[id * sc.segs + s]);
        }
        sum = (uint64_t)warp_sum_i64((int64_t)sum);
        first = __reduce_min_sync(0xffffffffu, first);
      }
      if (lane == 0) {
        sum_s[i] = sum;
        recip_s[i] = sum_recip(sum);
        first_s[i] = first;
      }
    }
    __syncthreads();
    // weights of the chunk: a warp takes eight rows and 32 keys at a time
    for (uint32_t u = warp; u < NT * steps; u += kTreeWarps) {
      const uint32_t n = u % NT, st = u / NT, i = 8 * n + (lane >> 2), f = f0 + i;
      int32_t x[8];
      int32_t total = 0;
      if (f < rows) {
        const size_t id = (size_t)(q.begin + f / q.group) * a.heads + g * q.group + f % q.group;
        const int32_t* s = sc.scores + id * sc.pitch + s0 + st * 32 + 4 * (lane & 3);
        const uint4 lo = *(const uint4*)s, hi = *(const uint4*)(s + 16);
        const uint32_t e[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        const uint32_t at = s0 + st * 32 + 4 * (lane & 3);
        weights_of(e, recip_s[i], sum_s[i], x);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          if (at + (j >> 2) * 16 + (j & 3) == first_s[i]) x[j] = 0;  // its weight comes last
          total += x[j];
        }
        total += __shfl_xor_sync(0xfu << (lane & 28), total, 1);
        total += __shfl_xor_sync(0xfu << (lane & 28), total, 2);
        if ((lane & 3) == 0 && total) atomicAdd(sc.wsum + id, total);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) x[j] = 0;
      }
      put_weight_fragment(w + (size_t)(st * NT + n) * 64, lane, x);
    }
    __syncthreads();
    // value sums: the warps take the head's 16-dimension tiles, and where
    // those are fewer than the warps, alternate steps of the keys
    const uint32_t tiles = a.head_dim / 16, split = max(1u, kTreeWarps / tiles);
    for (uint32_t u = warp; u < tiles * split; u += kTreeWarps) {
      const uint32_t dt = u % tiles, part = u / tiles;
      if (tree_value_tile<3>(a, sc, q, w, row_s, steps, g, f0, dt, part, split, lane))
        tree_value_tile<4>(a, sc, q, w, row_s, steps, g, f0, dt, part, split, lane);
    }
  }
  // the last block of this request and head writes the outputs
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    last_s = atom_add_acq_rel(sc.done + r * a.kv_heads + g, 1u) + 1 == chunks;
    __threadfence();
  }
  __syncthreads();
  if (!last_s) return;
  const size_t kvd = (size_t)a.kv_heads * a.head_dim;
  for (uint32_t f = warp; f < rows; f += kTreeWarps) {
    const uint32_t node = f / q.group, head = g * q.group + f % q.group;
    const size_t id = (size_t)(q.begin + node) * a.heads + head;
    uint32_t first = UINT32_MAX;
    for (uint32_t s = lane; s < segs; s += 32) first = min(first, sc.seg_first[id * sc.segs + s]);
    first = __reduce_min_sync(0xffffffffu, first);
    const int64_t row =
        first < q.count ? page_row(a.table + (size_t)r * a.width, a.width, a.page_size, a.pages, q.base + first) : -1;
    const int32_t top = sub_sat(kOneAct, __ldcg(sc.wsum + id));
    int32_t* out = a.out + (size_t)(q.begin + node) * a.out_stride + head * a.head_dim;
    for (uint32_t x = lane; x < a.head_dim; x += 32) {
      int64_t sum = __ldcg(sc.acc + id * a.head_dim + x);
      if (row >= 0) mac_wide(sum, top, a.v_pages[(size_t)row * kvd + g * a.head_dim + x]);
      out[x] = row >= 0 ? requantize(sum) : 0;
    }
  }
}

uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Keys a block takes: as many as leave the blocks enough for two a
// multiprocessor (fewer blocks reload fewer query fragments), at least 64.
uint32_t chunk_keys(const IrisTreeAttention& a) {
  const uint32_t groups = a.requests * a.kv_heads, want = 2 * 148;
  uint32_t chunk = 512;
  while (chunk > 64 && (uint64_t)groups * ceil_div(a.longest, chunk) < want) chunk /= 2;
  return chunk;
}

size_t carve(const IrisTreeAttention& a, uint8_t* base, TreeScratch* sc) {
  const size_t rows = (size_t)a.rows * a.heads;
  sc->chunk = chunk_keys(a);
  sc->chunks = ceil_div(a.longest, sc->chunk);
  sc->segs = ceil_div(a.longest, kTreeSegment);
  sc->pitch = ceil_div(a.longest, 64) * 64;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = base + at;
    at += up256(bytes);
    return p;
  };
  sc->scores = (int32_t*)take(rows * sc->pitch * 4);
  sc->chunk_max = (int32_t*)take(rows * sc->chunks * 4);
  sc->seg_sum = (uint64_t*)take(rows * sc->segs * 8);
  sc->seg_first = (uint32_t*)take(rows * sc->segs * 4);
  sc->acc = (int64_t*)take(rows * a.head_dim * 8);
  sc->wsum = (int32_t*)take(rows * 4);
  sc->done = (uint32_t*)take((size_t)a.requests * a.kv_heads * 4);
  return at;
}

constexpr uint32_t score_smem(uint32_t d) { return kTreeTile / 8 * (d / 32) * 4 * 256; }
constexpr uint32_t value_smem(uint32_t chunk) { return chunk / 32 * (kTreeTile / 8) * 512 + chunk * 8; }

}  // namespace

bool tree_mma_usable(const IrisTreeAttention& a) {
  return a.head_dim % 32 == 0 && a.scale_q32 < 0x80000000u && a.requests <= 65535 && a.kv_heads <= 65535 &&
         a.longest > 0;
}

uint64_t tree_mma_workspace(const IrisTreeAttention& a) {
  TreeScratch sc;
  return carve(a, nullptr, &sc);
}

cudaError_t launch_tree_mma(const IrisTreeAttention& a, uint8_t* workspace, cudaStream_t stream) {
  TreeScratch sc;
  carve(a, workspace, &sc);
  tree_scores_kernel<<<dim3(sc.chunks, a.kv_heads, a.requests), kTreeThreads, score_smem(a.head_dim), stream>>>(a, sc);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  e = launch_k(tree_terms_kernel, dim3(ceil_div(a.nodes * a.heads, kTreeWarps), sc.segs, a.requests),
               dim3(kTreeThreads), 0, stream, a, sc);
  if (e != cudaSuccess) return e;
  return launch_k(tree_values_kernel, dim3(sc.chunks, a.kv_heads, a.requests), dim3(kTreeThreads),
                  value_smem(sc.chunk), stream, a, sc);
}

}  // namespace iris
