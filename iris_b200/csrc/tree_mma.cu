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
// the keys' 512) stay in L2 between the launches while they fit.
// One node of sixteen requests over 4,000 keys (32 query heads, 8 of 128 values,
// 524 MB): 182 us, 2.9 TB/s of 6.46, the third launch 114 us (eight rows leave a
// product of 16 x 8 half used), the first 66: bound by the latency of reading K and
// V, of which a warp has one step of 32 dimensions or positions in flight ahead.
// 48 and 64 nodes over 20,011 and 32,001 keys: the second launch 184 us for 96 M
// exponentials, bound by their arithmetic (the same a pair where the scores fit L2).
#include <algorithm>

#include "../../include/iris_b200.h"
#include "common.cuh"
#include "layers.cuh"
#include "serve_attn.cuh"
#include "serve_mma.cuh"
#include "tree_mma.cuh"
#include "tree_tc.cuh"

namespace iris {

namespace {

constexpr uint32_t kTreeThreads = 256, kTreeWarps = kTreeThreads / 32;
__device__ __forceinline__ bool is_visible(const IrisTreeAttention& a, const TreeRequest& q, uint32_t node,
                                           uint32_t key) {
  const uint32_t row = q.begin + node;
  return tree_sees(key, q.held, (unsigned long long)a.masks[row] & node_bits(q.nodes), a.window,
                   a.positions ? (uint32_t)a.positions[row] : 0, a.positions + q.begin);
}

// 8 NT query rows at a time; with few rows more blocks share a multiprocessor,
// for their loads in flight.
template <uint32_t NT>
__global__ void __launch_bounds__(kTreeThreads, NT == 1 ? 4 : 2) tree_scores_kernel(IrisTreeAttention a, TreeScratch sc) {
  constexpr uint32_t kTreeTile = 8 * NT;
  extern __shared__ __align__(16) uint8_t tree_sm[];
  uint2* frag = (uint2*)tree_sm;  // [tile / 8][steps][4][32]
  __shared__ __align__(16) uint64_t row_at[kTreeTile];  // the rows' scores
  __shared__ uint32_t row_node[kTreeTile];
  __shared__ int32_t row_max[kTreeTile];
  __shared__ uint32_t q_wide;
  const uint32_t chunk = blockIdx.x, g = blockIdx.y, r = blockIdx.z;
  pdl_wait();
  if (sc.flags && !*sc.flags) return;  // the tensor-core launch did the work
  const TreeRequest q(a, r);
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, steps = a.head_dim / 32;
  const uint32_t rows = q.nodes * q.group, key0 = q.base + chunk * sc.chunk;
  if (chunk == 0 && !sc.flags) {  // the totals of this request and head start at zero
    for (uint32_t f = warp; f < rows; f += kTreeWarps) {
      const size_t id = (size_t)(q.begin + q.node_of(f)) * a.heads + q.head_of(f, g);
      for (uint32_t x = lane; x < a.head_dim; x += 32) sc.acc[id * a.head_dim + x] = 0;
      if (lane == 0) sc.wsum[id] = 0;
    }
    for (uint32_t i = tid; i < sc.groups; i += kTreeThreads) sc.done[((size_t)r * a.kv_heads + g) * sc.groups + i] = 0;
  }
  if (key0 >= q.keys) return;
  const uint32_t key1 = min(key0 + sc.chunk, q.base + (q.count + 15) / 16 * 16);
  const int32_t* table = a.table + (size_t)r * a.width;
  const size_t kvd = (size_t)a.kv_heads * a.head_dim;
  const QueryTile tile{frag, steps};
  for (uint32_t f0 = 0; f0 < rows; f0 += kTreeTile) {
    if (f0) __syncthreads();
    if (tid < kTreeTile) {
      // (rows past the last one repeat it)
      const uint32_t f = min(f0 + tid, rows - 1), node = q.node_of(f), head = q.head_of(f, g);
      row_node[tid] = node;
      row_at[tid] = ((size_t)(q.begin + node) * a.heads + head) * sc.pitch;
      row_max[tid] = INT32_MIN;
    }
    if (tid == 0) q_wide = 0;
    __syncthreads();
    for (uint32_t u = warp; u < NT * steps; u += kTreeWarps) {
      const uint32_t nt = u / steps, i = 8 * nt + (lane >> 2), f = min(f0 + i, rows - 1);
      const int32_t* src = a.q + (size_t)(q.begin + row_node[i]) * a.q_stride + q.head_of(f, g) * a.head_dim;
      if (put_query_fragment(frag, steps, nt, u % steps, lane, src)) q_wide = 1;
    }
    __syncthreads();
    const bool wide = q_wide != 0;
    int32_t best[NT][2];
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) best[n][0] = best[n][1] = INT32_MIN;
    for (uint32_t t0 = key0 + 16 * warp; t0 < key1; t0 += 16 * kTreeWarps) {
      const uint32_t ka = t0 + (lane >> 2), kb = ka + 8;
      const int64_t ra = ka < q.keys ? page_row(table, a.width, a.page_size, a.pages, ka) : -1;
      const int64_t rb = kb < q.keys ? page_row(table, a.width, a.page_size, a.pages, kb) : -1;
      const int32_t* pa = ra >= 0 ? a.k_pages + (size_t)ra * kvd + g * a.head_dim : nullptr;
      const int32_t* pb = rb >= 0 ? a.k_pages + (size_t)rb * kvd + g * a.head_dim : nullptr;
      // keys that every row sees need no look at the masks
      const bool open = t0 + 16 <= q.held && !a.window && __all_sync(0xffffffffu, ra >= 0 && rb >= 0);
      int32_t x[NT][4];
      key_scores<NT>(pa, pb, tile, wide, 0, lane, a.scale_q32, x);
      if (!open) {
#pragma unroll 1
        for (uint32_t u = 0; u < 2 * NT; ++u) {
          const uint32_t node = row_node[8 * (u / 2) + 2 * (lane & 3) + (u & 1)];
          const bool sa = ra >= 0 && is_visible(a, q, node, ka), sb = rb >= 0 && is_visible(a, q, node, kb);
#pragma unroll
          for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e)
              if (2 * n + e == u) {
                if (!sa) x[n][e] = INT32_MIN;
                if (!sb) x[n][e + 2] = INT32_MIN;
              }
        }
      }
      int32_t* out = sc.scores + (ka - q.base);
#pragma unroll
      for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) {
          int32_t* o = out + row_at[8 * n + 2 * (lane & 3) + e];
          o[0] = x[n][e];
          o[8] = x[n][e + 2];
          best[n][e] = max(best[n][e], max(x[n][e], x[n][e + 2]));
        }
    }
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e) {
        int32_t x = best[n][e];
#pragma unroll
        for (uint32_t o = 4; o <= 16; o <<= 1) x = max(x, __shfl_xor_sync(0xffffffffu, x, o));
        if (lane < 4) atomicMax(&row_max[8 * n + 2 * lane + e], x);
      }
    __syncthreads();
    if (tid < kTreeTile && f0 + tid < rows) sc.chunk_max[row_at[tid] / sc.pitch * sc.chunks + chunk] = row_max[tid];
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

// Rows f0 .. f0 + n - 1 of a request and K/V head: the totals, the first maximum's
// value times what the other weights leave of 1.0, rounded once. Rows that saw
// nothing give zeros.
__device__ __forceinline__ void finish_rows(const IrisTreeAttention& a, const int64_t* acc, const int32_t* wsum,
                                            const TreeRequest& q, const int32_t* table, uint32_t g, uint32_t f0,
                                            uint32_t n, const uint32_t* ids, const uint32_t* firsts, uint32_t warp,
                                            uint32_t warps, uint32_t lane) {
  const size_t kvd = (size_t)a.kv_heads * a.head_dim;
  for (uint32_t i = warp; i < n; i += warps) {
    const uint32_t node = q.node_of(f0 + i), head = q.head_of(f0 + i, g), first = firsts[i];
    const size_t id = ids[i];
    const int64_t row =
        first < q.count ? page_row(table, a.width, a.page_size, a.pages, q.base + first) : -1;
    const int32_t top = sub_sat(kOneAct, __ldcg(wsum + id));
    int32_t* out = a.out + (size_t)(q.begin + node) * a.out_stride + head * a.head_dim;
    for (uint32_t x = lane; x < a.head_dim; x += 32) {
      int64_t sum = __ldcg(acc + id * a.head_dim + x);
      if (row >= 0) mac_wide(sum, top, a.v_pages[(size_t)row * kvd + g * a.head_dim + x]);
      out[x] = row >= 0 ? requantize(sum) : 0;
    }
  }
}

// Values: a block takes up to 16 NT rows (8 NT for heads past 128 values) of one
// request and K/V head, and a chunk of its keys in stages of 64: the stage's
// values as byte-plane fragments and its weights go to shared memory, made once
// for all sixteen warps, which then take 16 dimensions x 8 NT rows each (where
// those are fewer than the warps, every other 32 keys too). The next stage's
// rows are in registers while this one's products run.
constexpr uint32_t kValueThreads = 512, kValueWarps = kValueThreads / 32, kValueKeys = 64;

struct ValueShared {
  uint64_t sum[64];
  uint32_t recip[64], first[64];
  uint32_t id[64];  // the rows' places in the scratch, UINT32_MAX past the last
  uint32_t wide, last;
};

template <uint32_t P, uint32_t NT>
__device__ __noinline__ bool tree_chunk_values(const IrisTreeAttention& a, const TreeScratch& sc, ValueShared& s,
                                               uint4* frag, uint2* wts, const uint32_t* row_s, uint32_t s0,
                                               uint32_t count, uint32_t g) {
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t dts = a.head_dim / 16, halves = dts <= 8 ? 2 : 1, units = dts * halves;
  const uint32_t split = units * 2 <= kValueWarps ? 2 : 1, unit = warp % units, part = warp / units;
  const uint32_t dt = unit % dts, half = unit / dts;
  const bool works = part < split;
  const size_t kvd = (size_t)a.kv_heads * a.head_dim;
  const uint32_t vfrags = dts * 2, wfrags = NT * halves * 2;  // fragments a stage
  const uint32_t stages = (count + kValueKeys - 1) / kValueKeys;
  int32_t acc[NT][P + 1][4];
#pragma unroll
  for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
    for (uint32_t d = 0; d < P + 1; ++d)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) acc[n][d][e] = 0;
  // this warp's fragments of a stage: values 16 wide u / 2, keys of half u & 1 (one
  // or, for wide heads, two), weights of rows 8 (u / 2) ..
  int2 x[8];
  uint4 t[2];
  const uint32_t wn = warp / 2, wst = warp & 1, wrow = 8 * wn + (lane >> 2);
  const bool weighs = warp < wfrags && s.id[wrow & 63] != UINT32_MAX;
  auto load_values = [&](uint32_t st, uint32_t u) {
    const int32_t* v = a.v_pages + g * a.head_dim + 16 * (u / 2) + 2 * (lane >> 2);
    const uint32_t* row = row_s + st * kValueKeys + (u & 1) * 32 + 4 * (lane & 3);
    const uint4 lo = *(const uint4*)row, hi = *(const uint4*)(row + 16);
    const uint32_t r[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) x[i] = *(const int2*)(v + (size_t)r[i] * kvd);
  };
  auto load_terms = [&](uint32_t st) {
    t[0] = t[1] = make_uint4(0, 0, 0, 0);
    const uint32_t at = st * kValueKeys + wst * 32;
    if (weighs && at < count) {
      const int32_t* e = sc.scores + (size_t)s.id[wrow] * sc.pitch + s0 + at + 4 * (lane & 3);
      t[0] = __ldcg((const uint4*)e);
      t[1] = __ldcg((const uint4*)(e + 16));
    }
  };
  uint32_t wide = 0;
  int32_t total = 0;
  if (warp < vfrags) load_values(0, warp);
  load_terms(0);
  for (uint32_t st = 0; st < stages; ++st) {
    uint4* fb = frag + (size_t)(st & 1) * vfrags * (P * 32);
    uint2* wb = wts + (size_t)(st & 1) * wfrags * 64;
    // fragments: [half of the keys][dimension tile], weights [half of the keys][row / 8]
    for (uint32_t u = warp; u < vfrags; u += kValueWarps) {
      if (u != warp) load_values(st, u);
      wide |= put_value_fragment<P>(fb + ((u & 1) * dts + u / 2) * (P * 32), x, lane);
    }
    if (warp < wfrags) {
      const uint32_t e[8] = {t[0].x, t[0].y, t[0].z, t[0].w, t[1].x, t[1].y, t[1].z, t[1].w};
      int32_t w[8];
      weights_of(e, weighs ? s.recip[wrow] : 0, s.sum[wrow & 63], w);
      const uint32_t at = s0 + st * kValueKeys + wst * 32 + 4 * (lane & 3), first = s.first[wrow & 63];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        if (at + (j >> 2) * 16 + (j & 3) == first) w[j] = 0;  // its weight comes last
        total += w[j];
      }
      put_weight_fragment(wb + (wst * (wfrags / 2) + wn) * 64, lane, w);
    }
    if (st + 1 < stages) {
      if (warp < vfrags) load_values(st + 1, warp);
      load_terms(st + 1);
    }
    __syncthreads();
    if (works)
      for (uint32_t h = part; h < 2; h += split)
        fragment_products<P, NT>(fb + (h * dts + dt) * (P * 32), wb + (h * (wfrags / 2) + half * NT) * 64, lane, acc);
  }
  if (P == 3) {
    if (wide) s.wide = 1;
    __syncthreads();
    if (s.wide) return true;
  }
  if (warp < wfrags) {
    total += __shfl_xor_sync(0xffffffffu, total, 1);
    total += __shfl_xor_sync(0xffffffffu, total, 2);
    if ((lane & 3) == 0 && weighs && total) atomicAdd(sc.wsum + s.id[wrow], total);
  }
  if (works) {
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t i = (half * NT + n) * 8 + 2 * (lane & 3) + (e & 1);
        if (s.id[i] != UINT32_MAX) {
          int32_t d[P + 1];
#pragma unroll
          for (uint32_t j = 0; j < P + 1; ++j) d[j] = acc[n][j][e];
          atomicAdd((unsigned long long*)(sc.acc + (size_t)s.id[i] * a.head_dim + 16 * dt + 2 * (lane >> 2) + (e >> 1)),
                    (unsigned long long)diagonal_sum(d));
        }
      }
  }
  return false;
}

template <uint32_t NT>
__global__ void __launch_bounds__(kValueThreads, 1) tree_values_kernel(IrisTreeAttention a, TreeScratch sc) {
  extern __shared__ __align__(16) uint8_t tree_sm[];
  __shared__ ValueShared s;
  if (sc.flags) {
    pdl_wait();
    if (!sc.flags[1]) return;  // the tensor-core launch did the work
  }
  const uint32_t dts = a.head_dim / 16, tile = 8 * NT * (dts <= 8 ? 2 : 1);  // rows
  const uint32_t groups = (a.nodes * (a.heads / a.kv_heads) + tile - 1) / tile;
  const uint32_t chunk = blockIdx.x, g = blockIdx.y / groups, f0 = blockIdx.y % groups * tile, r = blockIdx.z;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t* row_s = (uint32_t*)tree_sm;                    // [vchunk]: pool rows of the chunk's keys
  uint4* frag = (uint4*)(row_s + sc.vchunk);               // [2][2][dts][4][32]
  uint2* wts = (uint2*)(frag + (size_t)4 * dts * 4 * 32);  // [2][2][tile / 8][2][32]
  const TreeRequest q(a, r);
  const uint32_t rows = q.nodes * q.group, s0 = chunk * sc.vchunk, key0 = q.base + s0;
  const uint32_t chunks = (q.count + sc.vchunk - 1) / sc.vchunk, segs = (q.count + kTreeSegment - 1) / kTreeSegment;
  if (f0 >= rows || key0 >= q.keys) return;
  const uint32_t count = min(sc.vchunk, (q.keys - key0 + 31) / 32 * 32);
  const int32_t* table = a.table + (size_t)r * a.width;
  const uint32_t stand_in = stand_in_row(a, q, table);
  for (uint32_t i = tid; i < (count + kValueKeys - 1) / kValueKeys * kValueKeys; i += kValueThreads) {
    const int64_t row = key0 + i < q.keys ? page_row(table, a.width, a.page_size, a.pages, key0 + i) : -1;
    row_s[i] = row < 0 ? stand_in : (uint32_t)row;
  }
  if (tid == 0) s.wide = 0;
  if (!sc.flags) pdl_wait();
  for (uint32_t i = warp; i < tile; i += kValueWarps) {
    const uint32_t f = f0 + i;
    uint64_t sum = 0;
    uint32_t first = UINT32_MAX, id = UINT32_MAX;
    if (f < rows) {
      id = (q.begin + q.node_of(f)) * a.heads + q.head_of(f, g);
      for (uint32_t x = lane; x < segs; x += 32) {
        sum += sc.seg_sum[(size_t)id * sc.segs + x];
        first = min(first, sc.seg_first[(size_t)id * sc.segs + x]);
      }
      sum = (uint64_t)warp_sum_i64((int64_t)sum);
      first = __reduce_min_sync(0xffffffffu, first);
    }
    if (lane == 0) {
      s.sum[i] = sum;
      s.recip[i] = sum_recip(sum);
      s.first[i] = first;
      s.id[i] = id;
    }
  }
  __syncthreads();
  if (tree_chunk_values<3, NT>(a, sc, s, frag, wts, row_s, s0, count, g)) {
    __syncthreads();
    tree_chunk_values<4, NT>(a, sc, s, frag, wts, row_s, s0, count, g);
  }
  // the last block of these rows writes the outputs
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    s.last = atom_add_acq_rel(sc.done + (size_t)r * gridDim.y + blockIdx.y, 1u) + 1 == chunks;
    __threadfence();
  }
  __syncthreads();
  if (!s.last) return;
  finish_rows(a, sc.acc, sc.wsum, q, table, g, f0, min(tile, rows - f0), s.id, s.first, warp, kValueWarps, lane);
}

// Few rows (8 NT at most): values straight from their pages into the products, a
// chunk of keys a block of eight warps, so that several blocks a multiprocessor
// keep loads in flight: bound by reading the values.
template <uint32_t P, uint32_t NT>
__device__ __noinline__ bool few_values(const IrisTreeAttention& a, const TreeScratch& sc, const uint32_t* row_s,
                                        const uint2* w, const uint32_t* id_s, uint32_t part, uint32_t shares,
                                        uint32_t steps, uint32_t g, uint32_t dt, uint32_t lane) {
  const int32_t* v = a.v_pages + g * a.head_dim + 16 * dt + 2 * (lane >> 2);
  return paged_value_sums<P, NT>(v, (size_t)a.kv_heads * a.head_dim, row_s, w, part, shares, steps, lane,
                                 [&](uint32_t row, uint32_t x, int64_t sum) {
                                   if (id_s[row] != UINT32_MAX)
                                     atomicAdd((unsigned long long*)(sc.acc + (size_t)id_s[row] * a.head_dim + 16 * dt + x),
                                               (unsigned long long)sum);
                                 });
}

template <uint32_t NT>
__global__ void __launch_bounds__(kTreeThreads, 2)
    tree_few_values_kernel(IrisTreeAttention a, TreeScratch sc) {
  constexpr uint32_t R = 8 * NT;
  extern __shared__ __align__(16) uint8_t tree_sm[];
  uint32_t* row_s = (uint32_t*)tree_sm;         // [vchunk] pool rows
  uint2* wts = (uint2*)(row_s + sc.vchunk);     // [vchunk / 32][NT][2][32]
  __shared__ uint64_t sum_s[R];
  __shared__ uint32_t recip_s[R], first_s[R], id_s[R], last_s;
  __shared__ int32_t wsum_s[R];
  const uint32_t chunk = blockIdx.x, g = blockIdx.y, r = blockIdx.z;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const TreeRequest q(a, r);
  const uint32_t rows = q.nodes * q.group, s0 = chunk * sc.vchunk, key0 = q.base + s0;
  const uint32_t chunks = (q.count + sc.vchunk - 1) / sc.vchunk, segs = (q.count + kTreeSegment - 1) / kTreeSegment;
  if (!rows || key0 >= q.keys) return;
  const uint32_t count = min(sc.vchunk, (q.keys - key0 + 31) / 32 * 32), steps = count / 32;
  const int32_t* table = a.table + (size_t)r * a.width;
  const uint32_t stand_in = stand_in_row(a, q, table);
  for (uint32_t i = tid; i < count; i += kTreeThreads) {
    const int64_t row = key0 + i < q.keys ? page_row(table, a.width, a.page_size, a.pages, key0 + i) : -1;
    row_s[i] = row < 0 ? stand_in : (uint32_t)row;
  }
  if (tid < R) wsum_s[tid] = 0;
  pdl_wait();
#pragma unroll
  for (uint32_t i = warp; i < R; i += kTreeWarps) {
    uint64_t sum = 0;
    uint32_t first = UINT32_MAX, id = UINT32_MAX;
    if (i < rows) {
      id = (q.begin + q.node_of(i)) * a.heads + q.head_of(i, g);
      for (uint32_t x = lane; x < segs; x += 32) {
        sum += sc.seg_sum[(size_t)id * sc.segs + x];
        first = min(first, sc.seg_first[(size_t)id * sc.segs + x]);
      }
      sum = (uint64_t)warp_sum_i64((int64_t)sum);
      first = __reduce_min_sync(0xffffffffu, first);
    }
    if (lane == 0) {
      sum_s[i] = sum;
      recip_s[i] = sum_recip(sum);
      first_s[i] = first;
      id_s[i] = id;
    }
  }
  __syncthreads();
  for (uint32_t u = warp; u < NT * steps; u += kTreeWarps) {
    const uint32_t n = u % NT, st = u / NT, i = 8 * n + (lane >> 2), at = s0 + st * 32 + 4 * (lane & 3);
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    if (id_s[i] != UINT32_MAX) {
      const int32_t* t = sc.scores + (size_t)id_s[i] * sc.pitch + at;
      lo = __ldcg((const uint4*)t);
      hi = __ldcg((const uint4*)(t + 16));
    }
    const uint32_t e[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    int32_t w[8], all = 0;
    weights_of(e, recip_s[i], sum_s[i], w);
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      if (at + (j >> 2) * 16 + (j & 3) == first_s[i]) w[j] = 0;  // its weight comes last
      all += w[j];
    }
    put_weight_fragment(wts + (size_t)(st * NT + n) * 64, lane, w);
    all += __shfl_xor_sync(0xffffffffu, all, 1);
    all += __shfl_xor_sync(0xffffffffu, all, 2);
    if ((lane & 3) == 0 && all) atomicAdd(&wsum_s[i], all);
  }
  __syncthreads();
  const uint32_t dts = a.head_dim / 16, shares = max(1u, kTreeWarps / dts);  // warps a 16-dimension tile
  for (uint32_t u = warp; u < dts * shares; u += kTreeWarps)
    if (few_values<3, NT>(a, sc, row_s, wts, id_s, u / dts, shares, steps, g, u % dts, lane))
      few_values<4, NT>(a, sc, row_s, wts, id_s, u / dts, shares, steps, g, u % dts, lane);
  if (tid < R && id_s[tid] != UINT32_MAX && wsum_s[tid]) atomicAdd(sc.wsum + id_s[tid], wsum_s[tid]);
  // the last block of these rows writes the outputs
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    last_s = atom_add_acq_rel(sc.done + (size_t)r * gridDim.y + g, 1u) + 1 == chunks;
    __threadfence();
  }
  __syncthreads();
  if (last_s) finish_rows(a, sc.acc, sc.wsum, q, table, g, 0, min(R, rows), id_s, first_s, warp, kTreeWarps, lane);
}

uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Keys a block takes: as many as leave two blocks a multiprocessor (fewer
// blocks remake fewer query fragments), from 64 on.
uint32_t keys_a_block(uint64_t groups, uint32_t longest, uint32_t most, uint32_t want) {
  uint32_t chunk = most;
  while (chunk > 64 && groups * ceil_div(longest, chunk) < want) chunk /= 2;
  return chunk;
}

// The same for the tensor-core launches, whose blocks have a multiprocessor each
// and start with work of `start` tenths of a tile of 128 keys: one request is cut
// so that its blocks fill whole waves (sixty-four nodes over 12,000 keys: chunks of
// 128 keys 340 us, by this rule 223); several, whose lengths differ, into
// two waves or more.
uint32_t tc_keys_a_block(uint32_t requests, uint64_t groups, uint32_t longest, uint32_t start, uint32_t most) {
  if (requests > 1) return std::max(128u, keys_a_block(requests * groups, longest, most, 2 * 148));
  const uint32_t tiles = ceil_div(longest, 128), least = (uint32_t)((groups + 147) / 148);
  uint32_t best = 1;
  uint64_t cost = UINT64_MAX;
  for (uint32_t waves = least; waves < least + 8; ++waves) {
    const uint32_t t = std::min<uint64_t>(ceil_div(tiles, (uint32_t)std::min<uint64_t>(148 * waves / groups, tiles)), most / 128);
    const uint64_t blocks = groups * ceil_div(tiles, t), c = (blocks + 147) / 148 * (10 * t + start);
    if (c < cost) cost = c, best = t;
  }
  return best * 128;
}

// Row tiles a warp of the third launch takes (8 rows each, two warps a tile of
// dimensions for up to 128 of them): 32 rows do not pay for 64.
uint32_t value_tiles(const IrisTreeAttention& a) {
  return a.head_dim <= 128 && a.nodes * (a.heads / a.kv_heads) <= 32 ? 2 : 4;
}
// Row tiles of the first launch's blocks.
uint32_t score_tiles(const IrisTreeAttention& a) {
  const uint32_t rows = a.nodes * (a.heads / a.kv_heads);
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}
// Up to sixteen rows take their values straight from the pages.
bool few_rows(const IrisTreeAttention& a) { return a.nodes * (a.heads / a.kv_heads) <= 16; }
uint32_t value_rows(const IrisTreeAttention& a) { return value_tiles(a) * 8 * (a.head_dim <= 128 ? 2 : 1); }

size_t carve(const IrisTreeAttention& a, uint8_t* base, TreeScratch* sc) {
  const size_t rows = (size_t)a.rows * a.heads;
  sc->chunk = keys_a_block((uint64_t)a.requests * a.kv_heads, a.longest, 512, 2 * 148);
  if (tree_tc_usable(a))  // whole key tiles of the tensor-core launch
    sc->chunk = tc_keys_a_block(a.requests, a.kv_heads * ceil_div(a.nodes * (a.heads / a.kv_heads), kTreeTcRows), a.longest, 13, 4096);
  sc->chunks = ceil_div(a.longest, sc->chunk);
  sc->groups = few_rows(a) ? 1 : ceil_div(a.nodes * (a.heads / a.kv_heads), value_rows(a));
  sc->vchunk = few_rows(a) ? keys_a_block((uint64_t)a.requests * a.kv_heads, a.longest, 512, 4 * 148)
                           : keys_a_block((uint64_t)a.requests * a.kv_heads * sc->groups, a.longest, 4096, 2 * 148);
  sc->vchunks = ceil_div(a.longest, sc->vchunk);
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
  sc->done = (uint32_t*)take((size_t)a.requests * a.kv_heads * sc->groups * 4);
  sc->flags = nullptr;
  if (tree_tc_usable(a)) {
    sc->vchunk = 4096;  // (behind the tensor-core launch: few blocks to find that it did the work)
    sc->vchunks = ceil_div(a.longest, sc->vchunk);
    const uint32_t rows_most = a.nodes * (a.heads / a.kv_heads);
    sc->tc_rows = rows_most <= 64 ? 64 : 128;
    sc->tc_groups = ceil_div(rows_most, sc->tc_rows);
    sc->tc_vchunk = tc_keys_a_block(a.requests, (uint64_t)a.kv_heads * sc->tc_groups, a.longest, 20, 4096);
    sc->tc_vchunks = ceil_div(a.longest, sc->tc_vchunk);
    sc->tc_acc = (int64_t*)take(rows * a.head_dim * 8);
    sc->tc_wsum = (int32_t*)take(rows * 4);
    sc->tc_done = (uint32_t*)take((size_t)a.requests * a.kv_heads * sc->tc_groups * 4);
    sc->flags = (uint32_t*)take(8);
  }
  return at;
}

uint32_t score_smem(const IrisTreeAttention& a) { return score_tiles(a) * (a.head_dim / 32) * 4 * 256; }
constexpr uint32_t value_smem(uint32_t d, uint32_t vchunk, uint32_t rows) {
  return vchunk * 4 + 4 * (d / 16) * 4 * 512 + 4 * (rows / 8) * 512;
}

template <uint32_t NT>
cudaError_t launch_values(const IrisTreeAttention& a, const TreeScratch& sc, dim3 grid, uint32_t smem,
                          cudaStream_t stream) {
  static std::atomic<bool> allowed[64];
  const cudaError_t e = allow_smem(tree_values_kernel<NT>, allowed);
  if (e != cudaSuccess) return e;
  return launch_k(tree_values_kernel<NT>, grid, dim3(kValueThreads), smem, stream, a, sc);
}

}  // namespace

bool tree_mma_usable(const IrisTreeAttention& a) {
  return a.head_dim % 32 == 0 && a.scale_q32 < 0x80000000u && a.requests <= 65535 && a.kv_heads <= 65535 &&
         a.longest > 0 && a.longest <= 65535 * kTreeSegment && a.pages > 0 && a.pages * a.page_size < 0xFFFFFFFFull &&
         (uint64_t)a.rows * a.heads < 0xFFFFFFFFull && (uint64_t)a.heads * kTreeNodes <= 65535;
}

uint64_t tree_mma_workspace(const IrisTreeAttention& a) {
  TreeScratch sc;
  return carve(a, nullptr, &sc);
}

cudaError_t launch_tree_mma(const IrisTreeAttention& a, uint8_t* workspace, cudaStream_t stream) {
  TreeScratch sc;
  carve(a, workspace, &sc);
  cudaError_t e;
  if (sc.flags) {
    // totals, counters and flags, one behind another, start at zero
    e = cudaMemsetAsync(sc.acc, 0, (size_t)((uint8_t*)(sc.flags + 2) - (uint8_t*)sc.acc), stream);
    if (e == cudaSuccess) e = launch_tree_tc_scores(a, sc, stream);
    if (e != cudaSuccess) return e;
    e = launch_k(tree_scores_kernel<4>, dim3(sc.chunks, a.kv_heads, a.requests), dim3(kTreeThreads), score_smem(a),
                 stream, a, sc);
  } else {
    const dim3 grid(sc.chunks, a.kv_heads, a.requests);
    switch (score_tiles(a)) {
      case 1: tree_scores_kernel<1><<<grid, kTreeThreads, score_smem(a), stream>>>(a, sc); break;
      case 2: tree_scores_kernel<2><<<grid, kTreeThreads, score_smem(a), stream>>>(a, sc); break;
      default: tree_scores_kernel<4><<<grid, kTreeThreads, score_smem(a), stream>>>(a, sc); break;
    }
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  e = launch_k(tree_terms_kernel, dim3(ceil_div(a.nodes * a.heads, kTreeWarps), sc.segs, a.requests),
               dim3(kTreeThreads), 0, stream, a, sc);
  if (e == cudaSuccess && sc.flags) e = launch_tree_tc_values(a, sc, stream);
  if (e != cudaSuccess) return e;
  if (few_rows(a)) {
    const dim3 few(sc.vchunks, a.kv_heads, a.requests);
    const uint32_t few_smem = sc.vchunk * 4 + sc.vchunk / 32 * score_tiles(a) * 512;
    return score_tiles(a) == 1
               ? launch_k(tree_few_values_kernel<1>, few, dim3(kTreeThreads), few_smem, stream, a, sc)
               : launch_k(tree_few_values_kernel<2>, few, dim3(kTreeThreads), few_smem, stream, a, sc);
  }
  const uint32_t smem = value_smem(a.head_dim, sc.vchunk, value_rows(a));
  const dim3 grid(sc.vchunks, a.kv_heads * sc.groups, a.requests);
  return value_tiles(a) == 2 ? launch_values<2>(a, sc, grid, smem, stream)
                             : launch_values<4>(a, sc, grid, smem, stream);
}

}  // namespace iris
