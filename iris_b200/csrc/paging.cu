// Bookkeeping of a paged K/V cache that many requests share: the block tables
// and slot map of a step, K/V rows into their pages, and the acceptance of
// drafted tokens. Pages hold page_size token rows each; request r's token at
// position p lies in row (table[r][p / page_size] * page_size + p % page_size)
// of the pools.
#include <algorithm>

#include "../../include/iris_b200.h"
#include "common.cuh"
#include "serve.cuh"

namespace iris {

namespace {

// ---- the plan of a step -------------------------------------------------------
//
// offsets[r] = sum of fresh[0..r), and the new pages of request r are the
// entries [base[r], base[r + 1]) of the free list, base the prefix sums of
// ceil((held + fresh) / page) - ceil(held / page). Every block computes both
// prefix sums over all requests itself (the lengths are a few KB in L2; one
// coalesced round of loads and a scan in shared memory), so one launch needs no
// exchange between blocks; then it writes its share of the requests' offsets
// and table entries and of the tokens' slots. A warp finds its 32 tokens'
// first request by one search and steps on from there. Bound by latency: 32
// requests of 24 drafted tokens 5.5 us, 4,001 requests and a million tokens (12 MB)
// 15.3 us, about 5 of them the prefix sums.
constexpr uint32_t kPlanThreads = 512, kPlanWarps = kPlanThreads / 32;
constexpr uint32_t kPlanMaxRequests = 16384;  // two prefix sums and the lengths, 4 bytes a request each, in shared memory
constexpr uint32_t kPlanAhead = 4;            // tokens of a lane whose pages are read together

struct PlanArgs {
  const int32_t *held, *fresh, *free_pages, *parents;
  uint32_t requests, page, width, n_free, tokens;
  int32_t shift;  // log2 of the page size, -1 where it is no power of two
  uint32_t share; // tokens a block (a multiple of its threads)
  int32_t *table, *offsets, *positions, *counts;
  int64_t *slots, *masks;
};

__device__ __forceinline__ uint32_t page_of(uint32_t at, const PlanArgs& a) {
  return a.shift >= 0 ? at >> a.shift : at / a.page;
}
__device__ __forceinline__ uint32_t pages_of(uint32_t n, const PlanArgs& a) { return page_of(n + a.page - 1, a); }

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(PlanArgs a) {
  extern __shared__ uint32_t plan_sm[];
  uint32_t* off = plan_sm;                    // [requests + 1]
  uint32_t* base = plan_sm + a.requests + 1;  // [requests + 1]
  uint32_t* held = base + a.requests + 1;     // [requests]
  __shared__ unsigned long long part[kPlanWarps];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t bad = 0;
  // a request's tokens and new pages
#pragma unroll 4
  for (uint32_t r = tid; r < a.requests; r += kPlanThreads) {
    const int32_t h = a.held[r], f = a.fresh[r];
    const uint32_t hu = (uint32_t)max(h, 0), fu = (uint32_t)max(f, 0);
    if (h < 0 || f < 0 || hu + fu > (uint32_t)INT32_MAX) bad |= IRIS_PLAN_LENGTH;
    const uint32_t after = pages_of(hu + fu, a);
    if (after > a.width) bad |= IRIS_PLAN_WIDTH;
    off[r] = fu;
    held[r] = hu;
    base[r] = after - pages_of(hu, a);
  }
  __syncthreads();
  // prefix sums: a thread's run of consecutive requests, both sums in one word
  const uint32_t per = (a.requests + kPlanThreads - 1) / kPlanThreads;
  const uint32_t r0 = min(a.requests, tid * per), r1 = min(a.requests, r0 + per);
  uint64_t tok = 0, pg = 0;
  for (uint32_t r = r0; r < r1; ++r) tok += off[r], pg += base[r];
  const unsigned long long sum = ((unsigned long long)(uint32_t)tok << 32) | (uint32_t)pg;
  unsigned long long incl = sum;
#pragma unroll
  for (uint32_t d = 1; d < 32; d <<= 1) {
    const unsigned long long o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) part[warp] = incl;
  __syncthreads();
  unsigned long long before = incl - sum;
  for (uint32_t w = 0; w < warp; ++w) before += part[w];
  uint32_t t0 = (uint32_t)(before >> 32), p0 = (uint32_t)before;
  for (uint32_t r = r0; r < r1; ++r) {
    const uint32_t f = off[r], n = base[r];
    off[r] = t0;
    base[r] = p0;
    t0 += f;
    p0 += n;
    // (a request brings less than 2^31 tokens: the first sum past 31 bits shows; the
    // offsets wrap then, and what they index is checked all the same)
    if (t0 > (uint32_t)INT32_MAX) bad |= IRIS_PLAN_LENGTH;
  }
  if (r1 == a.requests && (r0 < r1 || (a.requests == 0 && tid == 0))) {
    off[a.requests] = t0;
    base[a.requests] = p0;
  }
  const uint32_t faults = (__syncthreads_or(bad & IRIS_PLAN_LENGTH) ? IRIS_PLAN_LENGTH : 0) |
                          (__syncthreads_or(bad & IRIS_PLAN_WIDTH) ? IRIS_PLAN_WIDTH : 0);
  const uint32_t total = off[a.requests], pages = base[a.requests];

  if (blockIdx.x == 0 && tid == 0) {
    a.counts[0] = (int32_t)total;
    a.counts[1] = (int32_t)pages;
    a.counts[2] = (int32_t)(total > a.tokens ? total - a.tokens : 0);
    a.counts[3] = (int32_t)(faults | (pages > a.n_free ? IRIS_PLAN_POOL : 0) | (total > a.tokens ? IRIS_PLAN_TOKENS : 0));
  }
  // the requests' offsets and new table entries: a block takes consecutive
  // requests, a thread a request's offset, a warp a request's entries
  const uint32_t span = (a.requests + gridDim.x) / gridDim.x;  // of requests + 1 offsets
  const uint32_t q0 = min(a.requests + 1, blockIdx.x * span), q1 = min(a.requests + 1, q0 + span);
  for (uint32_t r = q0 + tid; r < q1; r += kPlanThreads) a.offsets[r] = (int32_t)off[r];
  for (uint32_t r = q0 + warp; r < min(q1, a.requests); r += kPlanWarps) {
    const uint32_t n = base[r + 1] - base[r];
    if (!n) continue;
    const uint32_t first = pages_of(held[r], a);
    for (uint32_t j = lane; j < n && first + j < a.width; j += 32)
      a.table[(size_t)r * a.width + first + j] = base[r] + j < a.n_free ? a.free_pages[base[r] + j] : -1;
  }
  // the tokens' slots and positions: a warp's consecutive ones, kPlanAhead at a
  // time a lane, whose requests are steps from the last one's
  const uint32_t begin = blockIdx.x * a.share + warp * (a.share / kPlanWarps);
  const uint32_t end = min(a.tokens, begin + a.share / kPlanWarps);
  uint32_t r = begin < end && total ? request_of(off, a.requests, min(begin, total - 1)) : 0;
  for (uint32_t i0 = begin; i0 < end; i0 += 32 * kPlanAhead) {
    uint32_t own[kPlanAhead], at[kPlanAhead];
    int32_t id[kPlanAhead];
#pragma unroll
    for (uint32_t u = 0; u < kPlanAhead; ++u) {
      const uint32_t i = i0 + 32 * u + lane;
      id[u] = -1;
      at[u] = 0;
      if (i < min(total, end)) {
#pragma unroll
        for (uint32_t step = 0; step < 2; ++step) r += off[r + 1] <= i;
        if (off[r + 1] <= i) r += 1 + request_of(off + r + 1, a.requests - r - 1, i);
        at[u] = held[r] + i - off[r];
        const uint32_t column = page_of(at[u], a), first = pages_of(held[r], a);
        if (column < a.width) {
          const uint32_t fresh = base[r] + (column - first);
          if (column < first) id[u] = a.table[(size_t)r * a.width + column];
          else if (fresh < a.n_free) id[u] = a.free_pages[fresh];
        }
      }
      own[u] = r;
      r = __shfl_sync(0xffffffffu, r, 31);
    }
#pragma unroll
    for (uint32_t u = 0; u < kPlanAhead; ++u) {
      const uint32_t i = i0 + 32 * u + lane;
      if (i >= end) break;
      int64_t mask = 0;
      uint32_t position = at[u];
      if (a.masks && i < total && i - off[own[u]] < kTreeNodes) {
        // the node and its ancestors; a parent that is not an earlier node
        // (or a node past 64) leaves the mask empty
        const uint32_t first = off[own[u]];
        uint32_t node = i - first;
        unsigned long long m = 0;
        bool good = true;
        for (;;) {
          m |= 1ull << node;
          const int32_t up = a.parents[first + node];
          if (up == -1) break;
          if (up < 0 || (uint32_t)up >= node) {
            good = false;
            break;
          }
          node = (uint32_t)up;
        }
        if (good) {
          mask = (int64_t)m;
          position = held[own[u]] + (uint32_t)__popcll(m) - 1;
        }
      }
      a.slots[i] = id[u] < 0 ? -1 : (int64_t)id[u] * a.page + (at[u] - page_of(at[u], a) * a.page);
      a.positions[i] = (int32_t)position;
      if (a.masks) a.masks[i] = mask;
    }
  }
}

// ---- K/V rows into pages --------------------------------------------------------
//
// A copy: 16 bytes a thread and step, four loads in flight before their
// stores. Bound by memory (each row read once and written once): 8,191 rows of
// 1,024 values 21.8 us, 6.16 TB/s, 0.95 of a measured copy; 61 rows 2.6 us.
struct AppendArgs {
  const int32_t *k, *v;
  uint64_t k_stride, v_stride, rows;  // strides in values; rows of the pools
  uint32_t tokens, width4;            // a row's 16-byte pieces
  const int64_t* slots;
  int32_t *k_pages, *v_pages;
};

constexpr uint32_t kAppendThreads = 256, kAppendItems = 4;

__global__ void __launch_bounds__(kAppendThreads) page_append_kernel(AppendArgs a) {
  const uint64_t items = (uint64_t)a.tokens * a.width4;
  const int32_t* src = blockIdx.y ? a.v : a.k;
  int32_t* dst = blockIdx.y ? a.v_pages : a.k_pages;
  const uint64_t stride = blockIdx.y ? a.v_stride : a.k_stride;
  const uint64_t first = (uint64_t)blockIdx.x * (kAppendThreads * kAppendItems) + threadIdx.x;
  int4 x[kAppendItems];
  int64_t to[kAppendItems];
#pragma unroll
  for (uint32_t u = 0; u < kAppendItems; ++u) {
    const uint64_t i = first + u * kAppendThreads;
    to[u] = -1;
    if (i < items) {
      const uint32_t row = (uint32_t)(i / a.width4), c = (uint32_t)(i % a.width4);
      const int64_t slot = a.slots[row];
      if (slot >= 0 && (uint64_t)slot < a.rows) {
        to[u] = slot * a.width4 + c;
        x[u] = *(const int4*)(src + row * stride + 4 * (uint64_t)c);
      }
    }
  }
#pragma unroll
  for (uint32_t u = 0; u < kAppendItems; ++u)
    if (to[u] >= 0) ((int4*)dst)[to[u]] = x[u];
}

// ---- the acceptance of drafted tokens ---------------------------------------------
//
// From the root (node 0) the walk steps to the lowest child whose token is the
// pick at the current node, until there is none: a warp holds a request's 64
// nodes two a lane and finds each step with one ballot. The accepted nodes'
// K/V rows then move to the positions after the cached ones: node path[j]'s
// row to position held + j. path is increasing with path[j] >= j, so row j's
// target is never a later row's source: a column's rows may move in order of
// j with any number of loads ahead of the stores. Bound by latency: sixteen
// requests of 13 nodes in one layer 4.4 us, 48 of 61 in 32 layers (29 MB) 9.1 us,
// 3.2 TB/s.
struct AcceptArgs {
  const int32_t *tokens, *parents, *picks, *offsets, *held, *table;
  uint32_t requests, rows, width, page;  // rows: packed nodes of all requests
  int32_t *path, *accepted, *next, *held_out;
  uint32_t path_width;
  int32_t *k_pages, *v_pages;
  uint64_t layer_stride;  // values between two layers' pools
  uint64_t pages;
  uint32_t layers, kv4;   // a row's 16-byte pieces
};

constexpr uint32_t kAcceptThreads = 128, kAcceptAhead = 4;

__global__ void __launch_bounds__(kAcceptThreads) tree_accept_kernel(AcceptArgs a) {
  __shared__ uint32_t path[kTreeNodes];
  __shared__ int64_t from[kTreeNodes], to[kTreeNodes];
  __shared__ uint32_t moves_s;
  const uint32_t r = blockIdx.x, lane = threadIdx.x & 31;
  const uint32_t begin = clamp_offset(a.offsets[r], a.rows), stop = clamp_offset(a.offsets[r + 1], a.rows);
  const uint32_t n = min(stop > begin ? stop - begin : 0, min(kTreeNodes, a.path_width));
  const uint32_t held = (uint32_t)max(a.held[r], 0);
  if (threadIdx.x < 32) {
    int32_t up[2], token[2], pick[2];
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      const uint32_t i = lane + 32 * u;
      const bool in = i < n;
      up[u] = in ? a.parents[begin + i] : -1;
      token[u] = in ? a.tokens[begin + i] : 0;
      pick[u] = in ? a.picks[begin + i] : 0;
      if (!in || up[u] < 0 || up[u] >= (int32_t)i) up[u] = -2;  // node 0, and nodes that hang on nothing, are no child
    }
    uint32_t count = 0, at = 0;
    int32_t chosen = -1;
    while (count < n) {  // each step moves to a larger node: at most n of them
      if (lane == 0) path[count] = at;
      ++count;
      const int32_t p0 = __shfl_sync(0xffffffffu, pick[0], at & 31), p1 = __shfl_sync(0xffffffffu, pick[1], at & 31);
      chosen = at < 32 ? p0 : p1;
      const uint32_t b0 = __ballot_sync(0xffffffffu, up[0] == (int32_t)at && token[0] == chosen);
      const uint32_t b1 = __ballot_sync(0xffffffffu, up[1] == (int32_t)at && token[1] == chosen);
      if (!(b0 | b1)) break;
      at = b0 ? (uint32_t)__ffs(b0) - 1 : 32 + (uint32_t)__ffs(b1) - 1;
    }
    __syncwarp();
    if (blockIdx.y == 0) {
      for (uint32_t j = lane; j < a.path_width; j += 32)
        a.path[(size_t)r * a.path_width + j] = j < count ? (int32_t)path[j] : -1;
      if (lane == 0) {
        a.accepted[r] = (int32_t)count;
        a.next[r] = chosen;
        a.held_out[r] = (int32_t)(held + count);
      }
    }
    // the rows that move: a path's first nodes are in place while path[j] == j
    uint32_t moves = 0;
    if (a.k_pages) {
      for (uint32_t j0 = 0; j0 < count; j0 += 32) {
        const uint32_t j = j0 + lane;
        int64_t src = -1, dst = -1;
        if (j < count && path[j] != j) {
          src = page_row(a.table + (size_t)r * a.width, a.width, a.page, a.pages, held + path[j]);
          dst = page_row(a.table + (size_t)r * a.width, a.width, a.page, a.pages, held + j);
        }
        const uint32_t ok = __ballot_sync(0xffffffffu, src >= 0 && dst >= 0);
        if (ok >> lane & 1) {
          const uint32_t k = moves + (uint32_t)__popc(ok & ((1u << lane) - 1));
          from[k] = src * a.kv4;
          to[k] = dst * a.kv4;
        }
        moves += (uint32_t)__popc(ok);
      }
    }
    if (lane == 0) moves_s = moves;
  }
  __syncthreads();
  const uint32_t moves = moves_s;
  if (!moves) return;
  int4* pools[2] = {(int4*)(a.k_pages + blockIdx.y * a.layer_stride), (int4*)(a.v_pages + blockIdx.y * a.layer_stride)};
  for (uint32_t c = threadIdx.x; c < 2 * a.kv4; c += kAcceptThreads) {
    int4* pool = c < a.kv4 ? pools[0] : pools[1];
    const uint32_t column = c < a.kv4 ? c : c - a.kv4;
    for (uint32_t j = 0; j < moves; j += kAcceptAhead) {
      int4 x[kAcceptAhead];
#pragma unroll
      for (uint32_t u = 0; u < kAcceptAhead; ++u)
        if (j + u < moves) x[u] = pool[from[j + u] + column];
#pragma unroll
      for (uint32_t u = 0; u < kAcceptAhead; ++u)
        if (j + u < moves) pool[to[j + u] + column] = x[u];
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

}  // namespace iris

using namespace iris;

extern "C" {

int iris_page_plan(const int32_t* d_held, const int32_t* d_fresh, uint32_t requests, uint32_t page_size,
                   int32_t* d_table, uint32_t width, const int32_t* d_free, uint32_t n_free,
                   const int32_t* d_parents, uint32_t tokens, int32_t* d_offsets, int64_t* d_slots,
                   int32_t* d_positions, int64_t* d_masks, int32_t* d_counts, void* stream) {
  if (!d_offsets || !d_counts || !page_size || page_size > (1u << 20) || requests > kPlanMaxRequests ||
      tokens > (uint32_t)INT32_MAX || (requests && (!d_held || !d_fresh || (width && !d_table))) ||
      (n_free && !d_free) || (tokens && (!d_slots || !d_positions)) || (tokens && !d_parents != !d_masks))
    return IRIS_EINVAL;
  // two blocks a multiprocessor at most: each repeats the prefix sums
  const uint32_t rounds = (tokens + 2 * 148 * kPlanThreads - 1) / (2 * 148 * kPlanThreads);
  const uint32_t share = std::max(1u, rounds) * kPlanThreads;
  const int32_t shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  PlanArgs a{d_held, d_fresh, d_free, d_parents, requests, page_size, width, n_free, tokens, shift, share,
             d_table, d_offsets, d_positions, d_counts, d_slots, d_masks};
  const size_t smem = (size_t)(requests + 1) * 8 + (size_t)requests * 4;
  static std::atomic<bool> allowed[64];
  const cudaError_t e = allow_smem(page_plan_kernel, allowed);
  if (e != cudaSuccess) return (int)e;
  const uint32_t blocks = tokens ? (tokens + share - 1) / share : 1;
  page_plan_kernel<<<blocks, kPlanThreads, smem, (cudaStream_t)stream>>>(a);
  return (int)cudaGetLastError();
}

int iris_page_append(const int32_t* d_k, const int32_t* d_v, uint64_t k_stride, uint64_t v_stride, uint32_t tokens,
                     uint32_t kv_dim, const int64_t* d_slots, int32_t* d_k_pages, int32_t* d_v_pages,
                     uint64_t pool_rows, void* stream) {
  if (!kv_dim || kv_dim % 4 || kv_dim > (1u << 20) || pool_rows > ((uint64_t)1 << 40) || tokens > (uint32_t)INT32_MAX)
    return IRIS_EINVAL;
  if (!tokens) return 0;
  if (!d_k || !d_v || !d_slots || !d_k_pages || !d_v_pages || k_stride < kv_dim || v_stride < kv_dim ||
      k_stride % 4 || v_stride % 4 || !aligned16(d_k) || !aligned16(d_v) || !aligned16(d_k_pages) ||
      !aligned16(d_v_pages))
    return IRIS_EINVAL;
  AppendArgs a{d_k, d_v, k_stride, v_stride, pool_rows, tokens, kv_dim / 4, d_slots, d_k_pages, d_v_pages};
  const uint64_t items = (uint64_t)tokens * a.width4, per = kAppendThreads * kAppendItems;
  const uint64_t blocks = (items + per - 1) / per;
  if (blocks > (uint64_t)INT32_MAX) return IRIS_EINVAL;
  page_append_kernel<<<dim3((uint32_t)blocks, 2), kAppendThreads, 0, (cudaStream_t)stream>>>(a);
  return (int)cudaGetLastError();
}

int iris_tree_accept(const int32_t* d_tokens, const int32_t* d_parents, const int32_t* d_picks,
                     const int32_t* d_offsets, uint32_t requests, uint32_t rows, const int32_t* d_held,
                     uint32_t path_width, int32_t* d_path, int32_t* d_accepted, int32_t* d_next, int32_t* d_held_out,
                     const int32_t* d_table, uint32_t width, uint32_t page_size, int32_t* d_k_pages,
                     int32_t* d_v_pages, uint32_t layers, uint64_t layer_stride, uint64_t pages, uint32_t kv_dim,
                     void* stream) {
  if (!path_width || path_width > kTreeNodes || rows > (uint32_t)INT32_MAX || requests > (uint32_t)INT32_MAX ||
      !d_k_pages != !d_v_pages)
    return IRIS_EINVAL;
  if (!requests) return 0;
  if (!d_offsets || !d_held || !d_path || !d_accepted || !d_next || !d_held_out ||
      (rows && (!d_tokens || !d_parents || !d_picks)))
    return IRIS_EINVAL;
  if (d_k_pages) {
    if (!layers || layers > 65535 || !kv_dim || kv_dim % 4 || kv_dim > (1u << 20) || layer_stride % 4 || !page_size ||
        page_size > (1u << 20) || pages > ((uint64_t)1 << 31) || layer_stride < pages * page_size * kv_dim ||
        (width && !d_table) || !aligned16(d_k_pages) || !aligned16(d_v_pages))
      return IRIS_EINVAL;
  }
  AcceptArgs a{d_tokens, d_parents, d_picks, d_offsets, d_held, d_table, requests, rows, width, page_size,
               d_path, d_accepted, d_next, d_held_out, path_width, d_k_pages, d_v_pages, layer_stride, pages,
               layers, kv_dim / 4};
  tree_accept_kernel<<<dim3(requests, d_k_pages ? layers : 1), kAcceptThreads, 0, (cudaStream_t)stream>>>(a);
  return (int)cudaGetLastError();
}

}  // extern "C"
