// Drafted trees of few rows in one launch: plain decoding and small drafts,
// where latency counts.
//
// A thread-block cluster takes one request and K/V head; each of its blocks a
// span of the keys, whose scores, terms and weights stay in its shared memory.
// The blocks meet three times through distributed shared memory: the rows'
// maxima, the sums of their terms with the first maximum's place, and the value
// sums, which each block finishes for a share of the outputs. Keys and values
// are read once, straight into the matrix instructions' operands, and nothing
// goes through global memory but the outputs. Bound by latency on short
// contexts (three exchanges, two dependent reads of the pages: one node over 777
// keys, 32 query heads, 8 of 128 values, 14.7 us), by that of reading the pages on
// long ones, a step ahead in registers (four requests of one node over 12,000 keys
// 119 us, 3.3 TB/s of 6.46).
#include <cooperative_groups.h>

#include <algorithm>

#include "../../include/iris_b200.h"
#include "common.cuh"
#include "serve_mma.cuh"
#include "tree_cluster.cuh"
#include "tree_tc.cuh"

namespace iris {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kTcThreads = 256, kTcWarps = kTcThreads / 32;
constexpr uint32_t kClusterRows = 32;          // most rows

struct ClusterShared {
  int32_t top[kClusterRows];       // this block's, then the cluster's
  int32_t other_top[16][kClusterRows];
  unsigned long long sum[kClusterRows], other_sum[16][kClusterRows];
  uint32_t first[kClusterRows], other_first[16][kClusterRows];
  int32_t wsum[kClusterRows], other_wsum[16][kClusterRows];
  uint64_t total[kClusterRows];
  uint32_t recip[kClusterRows], at[kClusterRows], node[kClusterRows];
  uint32_t q_wide;
};

// cluster sums [row][d] of a warp's 16 dimensions.
template <uint32_t P, uint32_t NT>
__device__ __noinline__ bool cluster_values(const IrisTreeAttention& a, const uint32_t* row_s, const uint2* w,
                                            uint32_t steps, uint32_t g, uint32_t dt, int64_t* sums, uint32_t lane) {
  const int32_t* v = a.v_pages + g * a.head_dim + 16 * dt + 2 * (lane >> 2);
  return paged_value_sums<P, NT>(v, (size_t)a.kv_heads * a.head_dim, row_s, w, 0, 1, steps, lane,
                                 [&](uint32_t row, uint32_t x, int64_t sum) { sums[row * a.head_dim + 16 * dt + x] = sum; });
}

template <uint32_t NT>
__global__ void __launch_bounds__(kTcThreads) tree_cluster_kernel(IrisTreeAttention a, uint32_t span) {
  constexpr uint32_t R = 8 * NT;
  extern __shared__ __align__(16) uint8_t cl_sm[];
  __shared__ __align__(16) ClusterShared s;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const uint32_t g = blockIdx.y, r = blockIdx.z;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, steps = a.head_dim / 32;
  int32_t* scores = (int32_t*)cl_sm;                    // [R][span]: scores, terms
  int64_t* sums = (int64_t*)(scores + R * span);        // [R][head_dim]
  uint2* frag = (uint2*)(sums + R * a.head_dim);        // [NT][steps][4][32], then the weights [span / 32][NT][2][32]
  uint32_t* row_s = (uint32_t*)(frag + std::max(NT * steps * 128, span / 32 * NT * 64));  // [span] pool rows
  const TreeRequest q(a, r);
  const uint32_t rows = q.nodes * q.group;
  if (!rows) return;  // (of every block of the cluster)
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for before the first exchange)
  const uint32_t each = (q.count + ranks - 1) / ranks, mine = (each + 31) / 32 * 32;  // at most span
  const uint32_t s0 = rank * mine, count = s0 < q.count ? std::min(mine, q.count - s0) : 0, key0 = q.base + s0;
  const uint32_t padded = (count + 31) / 32 * 32;
  const int32_t* table = a.table + (size_t)r * a.width;
  const size_t kvd = (size_t)a.kv_heads * a.head_dim;
  const uint32_t stand_in = stand_in_row(a, q, table);
  for (uint32_t i = tid; i < padded; i += kTcThreads) {
    const int64_t row = i < count ? page_row(table, a.width, a.page_size, a.pages, key0 + i) : -1;
    row_s[i] = row < 0 ? UINT32_MAX : (uint32_t)row;
  }
  if (tid < R) {
    s.top[tid] = INT32_MIN;
    s.sum[tid] = 0;
    s.first[tid] = UINT32_MAX;
    s.wsum[tid] = 0;
    s.node[tid] = q.node_of(std::min(tid, rows - 1));
  }
  if (tid == 0) s.q_wide = 0;
  __syncthreads();
  for (uint32_t u = warp; u < NT * steps; u += kTcWarps) {
    const uint32_t nt = u / steps, f = std::min(8 * nt + (lane >> 2), rows - 1);  // (rows past the last repeat it)
    const int32_t* src = a.q + (size_t)(q.begin + q.node_of(f)) * a.q_stride + q.head_of(f, g) * a.head_dim;
    if (put_query_fragment(frag, steps, nt, u % steps, lane, src)) s.q_wide = 1;
  }
  __syncthreads();
  auto seen = [&](uint32_t row, uint32_t i) {
    return i < count && row_s[i] != UINT32_MAX && tree_sees(key0 + i, q.held, (unsigned long long)a.masks[q.begin + s.node[row]] & node_bits(q.nodes),
                     a.window, a.positions ? (uint32_t)a.positions[q.begin + s.node[row]] : 0,
                     a.positions + q.begin);
  };
  // scores
  const QueryTile tile{frag, steps};
  const bool q_wide = s.q_wide != 0;
  for (uint32_t t0 = 16 * warp; t0 < padded; t0 += 16 * kTcWarps) {
    const uint32_t ka = t0 + (lane >> 2), kb = ka + 8, ra = row_s[ka], rb = row_s[kb];
    const int32_t* pa = ra != UINT32_MAX ? a.k_pages + (size_t)ra * kvd + g * a.head_dim : nullptr;
    const int32_t* pb = rb != UINT32_MAX ? a.k_pages + (size_t)rb * kvd + g * a.head_dim : nullptr;
    const bool open = key0 + t0 + 16 <= q.held && !a.window && __all_sync(0xffffffffu, pa && pb);
    int32_t x[NT][4];
    key_scores<NT>(pa, pb, tile, q_wide, 0, lane, a.scale_q32, x);
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e) {
        const uint32_t i = 8 * n + 2 * (lane & 3) + e;
        int32_t y = x[n][e], z = x[n][e + 2];
        if (!open) {
          if (!seen(i, ka)) y = INT32_MIN;
          if (!seen(i, kb)) z = INT32_MIN;
        }
        scores[i * span + ka] = y;
        scores[i * span + kb] = z;
        int32_t m = std::max(y, z);
#pragma unroll
        for (uint32_t o = 4; o <= 16; o <<= 1) m = std::max(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane < 4) atomicMax(&s.top[i], m);
      }
  }
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every block runs
  // the rows' maxima over the cluster
  for (uint32_t i = tid; i < ranks * R; i += kTcThreads) {
    ClusterShared* peer = cluster.map_shared_rank(&s, i / R);
    peer->other_top[rank][i % R] = s.top[i % R];
  }
  cluster.sync();
  if (tid < R) {
    int32_t m = INT32_MIN;
    for (uint32_t b = 0; b < ranks; ++b) m = std::max(m, s.other_top[b][tid]);
    s.top[tid] = m;
  }
  __syncthreads();
  // terms: a warp a row and 32 keys a turn
  const uint32_t live = std::min(rows, R), parts = std::max(1u, kTcWarps / live);  // warps a row
  for (uint32_t u = warp; u < live * parts; u += kTcWarps) {
    const uint32_t i = u % live, part = u / live;
    const int32_t top = s.top[i];
    const bool ask = top < INT32_MIN + (1 << 20);
    uint64_t sum = 0;
    uint32_t first = UINT32_MAX;
    for (uint32_t t = part * 32 + lane; t < padded; t += parts * 32) {
      const uint32_t d = (uint32_t)top - (uint32_t)scores[i * span + t];
      uint32_t e = 0;
      if (d < kExpTerms) {
        bool doubt;
        e = exp_term_estimate(d, &doubt);
        if (doubt) e = d ? exp_term_near(d) : kTermTop;
        if (ask && !seen(i, t)) e = 0;
      }
      if (e == kTermTop) first = std::min(first, s0 + t);
      sum += kept_term(e);
      scores[i * span + t] = (int32_t)e;
    }
    sum = (uint64_t)warp_sum_i64((int64_t)sum);
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) {
      atomicAdd(&s.sum[i], (unsigned long long)sum);
      atomicMin(&s.first[i], first);
    }
  }
  __syncthreads();
  for (uint32_t i = tid; i < ranks * R; i += kTcThreads) {
    ClusterShared* peer = cluster.map_shared_rank(&s, i / R);
    peer->other_sum[rank][i % R] = s.sum[i % R];
    peer->other_first[rank][i % R] = s.first[i % R];
  }
  cluster.sync();
  if (tid < R) {
    uint64_t sum = 0;
    uint32_t first = UINT32_MAX;
    for (uint32_t b = 0; b < ranks; ++b) {
      sum += s.other_sum[b][tid];
      first = std::min(first, s.other_first[b][tid]);
    }
    if (tid >= live) sum = 0;  // (a row past the last one has no weights)
    s.total[tid] = sum;
    s.recip[tid] = sum_recip(sum);
    s.at[tid] = first;
  }
  for (uint32_t i = tid; i < padded; i += kTcThreads) row_s[i] = row_s[i] == UINT32_MAX ? stand_in : row_s[i];
  __syncthreads();
  // weights, over the query fragments
  for (uint32_t u = warp; u < NT * (padded / 32); u += kTcWarps) {
    const uint32_t n = u % NT, st = u / NT, i = 8 * n + (lane >> 2), at = st * 32 + 4 * (lane & 3);
    const uint4 lo = *(const uint4*)(scores + i * span + at), hi = *(const uint4*)(scores + i * span + at + 16);
    const uint32_t e[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    int32_t w[8], all = 0;
    weights_of(e, s.recip[i], s.total[i], w);
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      if (s0 + at + (j >> 2) * 16 + (j & 3) == s.at[i]) w[j] = 0;  // its weight comes last
      all += w[j];
    }
    put_weight_fragment(frag + (size_t)(st * NT + n) * 64, lane, w);
    all += __shfl_xor_sync(0xffffffffu, all, 1);
    all += __shfl_xor_sync(0xffffffffu, all, 2);
    if ((lane & 3) == 0 && all) atomicAdd(&s.wsum[i], all);
  }
  __syncthreads();
  if (padded) {
    for (uint32_t dt = warp; dt < a.head_dim / 16; dt += kTcWarps)
      if (cluster_values<3, NT>(a, row_s, frag, padded / 32, g, dt, sums, lane))
        cluster_values<4, NT>(a, row_s, frag, padded / 32, g, dt, sums, lane);
  } else {
    for (uint32_t i = tid; i < R * a.head_dim; i += kTcThreads) sums[i] = 0;
  }
  for (uint32_t i = tid; i < ranks * R; i += kTcThreads) {
    ClusterShared* peer = cluster.map_shared_rank(&s, i / R);
    peer->other_wsum[rank][i % R] = s.wsum[i % R];
  }
  cluster.sync();
  // this block's share of the outputs, from every block's sums
  const uint32_t outs = live * a.head_dim;
  for (uint32_t i = rank * kTcThreads + tid; i < outs; i += ranks * kTcThreads) {
    const uint32_t f = i / a.head_dim, x = i % a.head_dim;
    int64_t sum = 0;
    int32_t rest = kOneAct;
    for (uint32_t b = 0; b < ranks; ++b) {
      sum += cluster.map_shared_rank(sums, b)[i];
      rest -= s.other_wsum[b][f];
    }
    int32_t y = 0;
    if (s.at[f] != UINT32_MAX) {
      const int64_t row = page_row(table, a.width, a.page_size, a.pages, q.base + s.at[f]);
      mac_wide(sum, rest, a.v_pages[(size_t)row * kvd + g * a.head_dim + x]);
      y = requantize(sum);
    }
    a.out[(size_t)(q.begin + q.node_of(f)) * a.out_stride + q.head_of(f, g) * a.head_dim + x] = y;
  }
  cluster.sync();  // the others' reads of this block's sums are over
}

uint32_t row_tiles(const IrisTreeAttention& a) {
  const uint32_t rows = a.nodes * (a.heads / a.kv_heads);
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}
// Blocks a multiprocessor holds: two of up to eight rows; more rows' registers
// allow no second.
uint32_t blocks_a_sm(const IrisTreeAttention& a) { return row_tiles(a) == 1 ? 2 : 1; }
// Blocks of a cluster: as many as are on the device at once, and 32 keys a
// block. A cluster's blocks lie together, so that fifteen clusters of eight blocks
// a multiprocessor each find room, 33 of four, 74 of two; two blocks a
// multiprocessor 33, 71 and 148 (four drafts of sixteen requests over 777 keys, 4
// query heads of 64: sixteen clusters of eight 30.7 us, of four 20.1; one node of
// four requests over 4,000 keys, 32 heads and 8 of 128: 32 clusters of eight 49 us,
// of four 74). Sixteen only for up to eight rows on a free device: of many such
// clusters few are free in one place (33 against 22 us for sixteen requests of 777
// keys).
uint32_t cluster_blocks(const IrisTreeAttention& a) {
  const uint64_t groups = (uint64_t)a.requests * a.kv_heads;
  const bool two = blocks_a_sm(a) == 2;
  if (two && groups * 16 <= 148 && 15 * 32 < a.longest) return 16;
  const auto room = [&](uint32_t n) { return n == 8 ? (two ? 33u : 15u) : n == 4 ? (two ? 71u : 33u) : (two ? 148u : 74u); };
  uint32_t n = 8;
  while (n > 1 && (groups > room(n) || (n - 1) * 32 >= a.longest)) n /= 2;
  return n;
}
uint32_t block_span(const IrisTreeAttention& a) {
  const uint32_t n = cluster_blocks(a), each = (a.longest + n - 1) / n;
  return (each + 31) / 32 * 32;
}

template <uint32_t NT>
cudaError_t launch(const IrisTreeAttention& a, cudaStream_t stream) {
  static std::atomic<bool> allowed[64], wide_clusters[64];
  cudaError_t e = allow_smem(tree_cluster_kernel<NT>, allowed);
  if (e != cudaSuccess) return e;
  const uint32_t span = block_span(a), steps = a.head_dim / 32, R = 8 * NT;
  const uint32_t smem = R * span * 4 + R * a.head_dim * 8 + std::max(NT * steps * 128, span / 32 * NT * 64) * 8 + span * 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster_blocks(a), a.kv_heads, a.requests);
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cfg.gridDim.x;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cfg.gridDim.x > 8) {
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!wide_clusters[dev].load(std::memory_order_acquire)) {
      e = cudaFuncSetAttribute(tree_cluster_kernel<NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return e;
      wide_clusters[dev].store(true, std::memory_order_release);
    }
  }
  return cudaLaunchKernelEx(&cfg, tree_cluster_kernel<NT>, a, span);
}

}  // namespace

// Few rows, and spans of keys that a block is done with before the three launches
// of tree_mma.cu are: up to 256; where the blocks fill much of the device, all at
// once, up to 1,536 for eight rows, 1,024 for sixteen, 512 for more. Measured, us,
// here against there: 32 query heads, 8 K/V heads of 128: one node over 777 keys
// 14.8 / 20.7, over 8,000 35 / 54, over 30,000 242 / 106; four requests over
// 12,000 119 / 147, sixteen over 2,000 86 / 107, over 4,000 264 / 181, forty over
// 777 130 / 118; four nodes over 8,000 64 / 84; eight nodes over 777 24.3 / 38.3,
// four requests of them over 2,000 58 / 96. 8 query heads, 1 K/V head of 256: one
// node over 4,000 25.1 / 24.6, over 8,000 39.5 / 26.9; four over 4,000 71 / 42,
// eight requests of them 85 / 129.
bool tree_cluster_usable(const IrisTreeAttention& a) {
  const uint32_t rows = a.nodes * (a.heads / a.kv_heads);
  if (rows > kClusterRows) return false;
  const uint32_t tiles = row_tiles(a), span = block_span(a), most = tiles == 1 ? 1536 : tiles == 2 ? 1024 : 512;
  const uint64_t blocks = (uint64_t)a.requests * a.kv_heads * cluster_blocks(a);
  return span <= 256 || (span <= most && blocks >= 64 && blocks <= 148 * blocks_a_sm(a));
}

cudaError_t launch_tree_cluster(const IrisTreeAttention& a, cudaStream_t stream) {
  switch (row_tiles(a)) {
    case 1: return launch<1>(a, stream);
    case 2: return launch<2>(a, stream);
    default: return launch<4>(a, stream);
  }
}

}  // namespace iris
