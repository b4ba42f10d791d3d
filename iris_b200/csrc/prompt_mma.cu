// Packed prompt attention on the matrix instructions.
//
// A persistent block takes one tile of query rows at a time: RT consecutive
// rows of one request that share a K/V head (the query heads of a group are
// neighbouring rows, so a key is fetched once for all of them), with the keys
// they see, in three phases over them:
//   1. scores into a scratch of the block's own, and the rows' maxima;
//   2. the exponentials in place, a row a warp: sums and first maxima;
//   3. weights, 128 keys at a time through shared memory, and the value sums.
// The integer softmax needs a row's exact sum before its first weight, so the
// scores are kept: 4 bytes a row and key, written and read by one block within
// its item, which mostly stays in L2. Tiles are handed out longest first; few
// tiles, a block each, are counted by the blocks themselves in one launch.
// Bound by the chain of its phases on a few rows (five requests of up to 96 rows, 4
// heads of 64, 27 us on thirteen blocks; with the list in a launch of its own 39 us) and by the products and the score and
// exponential arithmetic on many (512 rows, 32 heads of 128, 101 us; prompt_tc.cu
// takes over there).
#include <algorithm>

#include "../../include/iris_b200.h"
#include "common.cuh"
#include "layers.cuh"
#include "prompt_mma.cuh"
#include "prompt_tc.cuh"
#include "serve_attn.cuh"
#include "serve_mma.cuh"
#include "tc.cuh"

namespace iris {

namespace {

constexpr uint32_t kPromptThreads = 512, kPromptWarps = kPromptThreads / 32;
constexpr uint32_t kPromptKeys = 128;  // keys of a weight tile
constexpr uint32_t kSortRequests = 1024;
constexpr uint32_t kFewRequests = 32;  // whose tiles a block counts itself, with 148 blocks' worth of tiles at most

struct PromptScratch {
  uint32_t* order;   // [requests]: the requests, longest first
  uint32_t* tiles;   // [requests + 1]: tiles before each of them
  uint32_t* tc_tiles;  // the same for prompt_tc_kernel's tiles
  uint32_t* next;    // the item counters of this kernel and of prompt_tc_kernel
  int32_t* scores;   // [blocks][RT][pitch]
  int64_t* acc;      // [blocks][RT][d]: value sums, where several warps or segments add to one
  uint32_t pitch, blocks;
  const uint32_t* wide;  // [flags]: with the tensor-core kernel before this one, whether it left the call to it
  uint32_t flags;
};

// The tiles of each request, longest first (up to 1024 requests; more keep
// their order), and the item counters. The second block, where there is one,
// counts the tensor-core kernel's tiles of 64 rows.
__global__ void __launch_bounds__(1024) prompt_items_kernel(IrisPromptAttention a, PromptScratch sc, uint32_t rt) {
  __shared__ int32_t len_s[kSortRequests];
  __shared__ uint32_t part[32];
  __shared__ uint32_t carry;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.heads / a.kv_heads;
  auto length = [&](uint32_t r) {
    const uint32_t b = clamp_offset(a.offsets[r], a.tokens), e = clamp_offset(a.offsets[r + 1], a.tokens);
    return e > b ? min(e - b, a.longest) : 0u;
  };
  pdl_trigger();
  uint32_t* tiles = blockIdx.x ? sc.tc_tiles : sc.tiles;
  if (blockIdx.x) rt = 64;
  if (tid == 0) {
    sc.next[blockIdx.x] = 0;
    carry = 0;
  }
  const bool sorted = a.requests <= kSortRequests;
  if (sorted) {
    if (tid < a.requests) len_s[tid] = (int32_t)length(tid);
    __syncthreads();
    if (tid < a.requests) {
      uint32_t rank = 0;
      for (uint32_t r = 0; r < a.requests; ++r) rank += len_s[r] > len_s[tid] || (len_s[r] == len_s[tid] && r < tid);
      sc.order[rank] = tid;
    }
  } else {
    for (uint32_t r = tid; r < a.requests; r += 1024) sc.order[r] = r;
  }
  __syncthreads();
  for (uint32_t r0 = 0; r0 < a.requests; r0 += 1024) {
    const uint32_t r = r0 + tid;
    const uint32_t n =
        r < a.requests ? (uint32_t)(((uint64_t)length(sc.order[r]) * group + rt - 1) / rt) : 0;
    uint32_t incl = n;
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    if (lane == 31) part[warp] = incl;
    __syncthreads();
    uint32_t before = carry + incl - n;
    for (uint32_t w = 0; w < warp; ++w) before += part[w];
    if (r < a.requests) tiles[r] = before;
    __syncthreads();
    if (tid == 1023) carry = before + n;
    __syncthreads();
  }
  if (tid == 0) tiles[a.requests] = carry;
}

// One tile: rows f0 .. f0 + RT - 1 of a request's len * group rows (row f is
// query f / group, head f % group of the K/V head), and its keys.
struct PromptTile {
  uint32_t begin, len, group, g, f0, rows, base, count;
};

// Value sums of one warp's unit (16 dimensions x 32 rows) over weight steps
// [0, steps) of a tile in shared memory.
template <uint32_t P>
__device__ __forceinline__ uint32_t prompt_value_steps(const IrisPromptAttention& a, const PromptTile& p,
                                                       const uint2* w, uint32_t row_tiles, uint32_t key,
                                                       uint32_t first, uint32_t by, uint32_t steps, uint32_t dt,
                                                       uint32_t lane, int32_t (&acc)[4][P + 1][4]) {
  const int32_t* v = a.v + (uint64_t)p.begin * a.v_stride + p.g * a.head_dim + 16 * dt + 2 * (lane >> 2);
  const uint32_t end = p.base + p.count - 1;
  int2 x[8];
  auto load = [&](uint32_t st) {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t t = min(end, key + st * 32 + (i >> 2) * 16 + 4 * (lane & 3) + (i & 3));  // weights past it are 0
      x[i] = *(const int2*)(v + (uint64_t)t * a.v_stride);
    }
  };
  uint32_t wide = 0;
  for (uint32_t st = first; st < steps; st += by) {
    load(st);
    wide |= value_products<P, 4>(x, w + (uint64_t)st * row_tiles * 64, lane, acc);
  }
  return wide;
}

template <uint32_t RT>
struct PromptShared {
  int32_t top[RT];
  int32_t query[RT];  // the row's query, -1 past the last row
  uint64_t sum[RT];
  uint32_t recip[RT], first[RT];
  int32_t wsum[RT];
  uint32_t wide, item;
};

// Phase 3 with P value planes; returns whether a value was past 24 bits (P = 3:
// nothing was written then).
template <uint32_t RT, uint32_t P>
__device__ __noinline__ bool prompt_values(const IrisPromptAttention& a, const PromptTile& p, PromptShared<RT>& s,
                                           uint2* w, const int32_t* scores, uint32_t pitch, int64_t* acc_buf) {
  constexpr uint32_t NT = RT / 8;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t dts = a.head_dim / 16, units = dts * (RT / 32), split = max(1u, kPromptWarps / units);
  const uint32_t unit = warp % units, part = warp / units, dt = unit % dts, half = unit / dts;
  const bool works = part < split, shared_acc = split > 1 || p.count > kPvKeys;
  if (shared_acc)
    for (uint32_t i = tid; i < RT * a.head_dim; i += kPromptThreads) acc_buf[i] = 0;
  if (tid < RT) s.wsum[tid] = 0;
  if (tid == 0) s.wide = 0;
  __syncthreads();
  int32_t acc[4][P + 1][4];
  auto clear = [&] {
#pragma unroll
    for (uint32_t n = 0; n < 4; ++n)
#pragma unroll
      for (uint32_t d = 0; d < P + 1; ++d)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) acc[n][d][e] = 0;
  };
  auto total = [&](uint32_t n, uint32_t e) {
    int32_t d[P + 1];
#pragma unroll
    for (uint32_t j = 0; j < P + 1; ++j) d[j] = acc[n][j][e];
    return diagonal_sum(d);
  };
  auto flush = [&] {
#pragma unroll
    for (uint32_t n = 0; n < 4; ++n)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        atomicAdd((unsigned long long*)acc_buf + (half * 32 + 8 * n + 2 * (lane & 3) + (e & 1)) * a.head_dim + 16 * dt +
                      2 * (lane >> 2) + (e >> 1),
                  (unsigned long long)total(n, e));
  };
  clear();
  uint32_t wide = 0, buf = 0;
  for (uint32_t t0 = 0; t0 < p.count; t0 += kPromptKeys, buf ^= 1) {
    const uint32_t steps = min(kPromptKeys, p.count - t0 + 31) / 32;
    uint2* wb = w + (uint64_t)buf * (kPromptKeys / 32) * NT * 64;
    for (uint32_t u = warp; u < NT * steps; u += kPromptWarps) {
      const uint32_t n = u % NT, st = u / NT, i = 8 * n + (lane >> 2);
      const int32_t* e = scores + (uint64_t)i * pitch + t0 + st * 32 + 4 * (lane & 3);
      const uint4 lo = __ldcg((const uint4*)e), hi = __ldcg((const uint4*)(e + 16));
      const uint32_t term[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      const uint32_t recip = s.recip[i];
      const uint64_t sum = s.sum[i];
      int32_t x[8], all = 0;
      weights_of(term, recip, sum, x);
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) all += x[j];
      put_weight_fragment(wb + (st * NT + n) * 64, lane, x);
      all += __shfl_xor_sync(0xffffffffu, all, 1);
      all += __shfl_xor_sync(0xffffffffu, all, 2);
      if ((lane & 3) == 0 && all) atomicAdd(&s.wsum[i], all);
    }
    __syncthreads();  // (two buffers: the next tile's weights are written while this one's are read)
    if (works) {
      wide |= prompt_value_steps<P>(a, p, wb + half * 4 * 64, NT, p.base + t0, part, split, steps, dt, lane, acc);
      if (shared_acc && (t0 + kPromptKeys) % kPvKeys == 0) {
        flush();
        clear();
      }
    }
  }
  if (P == 3 && wide) s.wide = 1;
  if (shared_acc && works) flush();
  __syncthreads();
  if (P == 3 && s.wide) {
    __syncthreads();
    return true;
  }
  auto write = [&](uint32_t i, uint32_t x, int64_t s0, int64_t s1) {  // row i, dimensions x and x + 1
    const uint32_t f = p.f0 + i;
    const int32_t wt = sub_sat(kOneAct, s.wsum[i]);
    const int2 v = *(const int2*)(a.v + (uint64_t)(p.begin + p.base + s.first[i]) * a.v_stride + p.g * a.head_dim + x);
    mac_wide(s0, wt, v.x);
    mac_wide(s1, wt, v.y);
    *(int2*)(a.out + (uint64_t)(p.begin + f / p.group) * a.out_stride + (p.g * p.group + f % p.group) * a.head_dim +
             x) = make_int2(requantize(s0), requantize(s1));
  };
  if (shared_acc) {
    for (uint32_t i = tid; i < p.rows * (a.head_dim / 2); i += kPromptThreads) {
      const uint32_t row = i / (a.head_dim / 2), x = i % (a.head_dim / 2) * 2;
      write(row, x, __ldcg(acc_buf + row * a.head_dim + x), __ldcg(acc_buf + row * a.head_dim + x + 1));
    }
  } else if (works) {
#pragma unroll
    for (uint32_t n = 0; n < 4; ++n)
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e) {
        const uint32_t i = half * 32 + 8 * n + 2 * (lane & 3) + e;
        if (i < p.rows) write(i, 16 * dt + 2 * (lane >> 2), total(n, e), total(n, e + 2));
      }
  }
  return false;
}

template <uint32_t RT>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt_mma_kernel(IrisPromptAttention a, PromptScratch sc) {
  constexpr uint32_t NT = RT / 8;
  extern __shared__ __align__(16) uint8_t prompt_sm[];
  __shared__ PromptShared<RT> s;
  const uint32_t steps = a.head_dim / 32;
  uint2* frag = (uint2*)prompt_sm;                  // [NT][steps][4][32]
  uint2* w = frag + NT * steps * 128;               // [2][kPromptKeys / 32][NT][2][32]
  uint32_t* lists = (uint32_t*)(w + 2 * kPromptKeys / 32 * NT * 64);  // [warps][kTermList]
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* scores = sc.scores + (uint64_t)blockIdx.x * RT * sc.pitch;
  int64_t* acc_buf = sc.acc + (uint64_t)blockIdx.x * RT * a.head_dim;
  const QueryTile tile{frag, steps};
  pdl_wait();
  pdl_trigger();
  if (sc.flags) {
    uint32_t wide = 0;
    for (uint32_t i = tid; i < sc.flags; i += kPromptThreads) wide |= sc.wide[i];
    if (!__syncthreads_or(wide != 0)) return;
  }
  // Few requests: every block counts the tiles itself, and takes every so manyth
  // of them; else the list of prompt_items_kernel, handed out one by one.
  __shared__ uint32_t few_tiles[kFewRequests + 1];
  const bool few = sc.order == nullptr;
  if (few && warp == 0) {
    uint32_t n = 0;
    if (lane < a.requests) {
      const uint32_t b = clamp_offset(a.offsets[lane], a.tokens), e = clamp_offset(a.offsets[lane + 1], a.tokens);
      n = e > b ? (uint32_t)(((uint64_t)min(e - b, a.longest) * (a.heads / a.kv_heads) + RT - 1) / RT) : 0;
    }
    uint32_t incl = n;
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    few_tiles[lane] = incl - n;
    if (lane == 31) few_tiles[kFewRequests] = incl;
  }
  __syncthreads();
  const uint32_t* tiles = few ? few_tiles : sc.tiles;
  const uint32_t items = (few ? few_tiles[kFewRequests] : sc.tiles[a.requests]) * a.kv_heads;
  for (uint32_t mine = blockIdx.x;; mine += gridDim.x) {
    __syncthreads();  // the tile before is done with the shared memory
    if (!few && tid == 0) s.item = atomicAdd(sc.next, 1u);
    __syncthreads();
    const uint32_t item = few ? mine : s.item;
    if (item >= items) return;
    PromptTile p;
    p.g = item % a.kv_heads;
    const uint32_t at = item / a.kv_heads, rank = request_of(tiles, few ? kFewRequests : a.requests, at);
    const uint32_t r = few ? rank : sc.order[rank];
    p.begin = clamp_offset(a.offsets[r], a.tokens);
    p.len = min(clamp_offset(a.offsets[r + 1], a.tokens) - p.begin, a.longest);
    p.group = a.heads / a.kv_heads;
    p.f0 = (tiles[rank + 1] - 1 - at) * RT;  // a request's last tile, the longest, first
    p.rows = min(RT, p.len * p.group - p.f0);
    const uint32_t q0 = p.f0 / p.group, q1 = (p.f0 + p.rows - 1) / p.group;
    p.base = window_start(q0, a.window) / 16 * 16;
    p.count = q1 + 1 - p.base;

    // the query rows as fragments
    if (tid < RT) {
      s.top[tid] = INT32_MIN;
      s.query[tid] = tid < p.rows ? (int32_t)((p.f0 + tid) / p.group) : -1;
    }
    if (tid == 0) s.wide = 0;
    __syncthreads();
    for (uint32_t u = warp; u < NT * steps; u += kPromptWarps) {
      const uint32_t nt = u / steps, i = 8 * nt + (lane >> 2);
      const int32_t* src = nullptr;
      if (i < p.rows)
        src = a.q + (uint64_t)(p.begin + s.query[i]) * a.q_stride +
              (p.g * p.group + (p.f0 + i) % p.group) * a.head_dim;
      if (put_query_fragment(frag, steps, nt, u % steps, lane, src)) s.wide = 1;
    }
    __syncthreads();

    // 1. scores, 16 keys x 32 rows a warp and turn; hidden ones carry the lowest score
    const bool q_wide = s.wide != 0;
    const int32_t* k = a.k + (uint64_t)p.begin * a.k_stride + p.g * a.head_dim;
    const uint32_t last_key = p.base + p.count - 1;
    for (uint32_t u = warp; u / (NT / 4) * 16 < p.count; u += kPromptWarps) {
      const uint32_t t0 = u / (NT / 4) * 16, nt0 = u % (NT / 4) * 4;
      const uint32_t ka = p.base + t0 + (lane >> 2), kb = ka + 8;
      const int32_t* pa = k + (uint64_t)min(ka, last_key) * a.k_stride;
      const int32_t* pb = k + (uint64_t)min(kb, last_key) * a.k_stride;
      // keys that every row sees
      const bool open = p.base + t0 + 15 <= q0 && (!a.window || p.base + t0 >= window_start(q1, a.window));
      int32_t x[4][4];
      key_scores<4>(pa, pb, tile, q_wide, nt0, lane, a.scale_q32, x);
      int32_t* out = scores + (uint64_t)(8 * nt0 + 2 * (lane & 3)) * sc.pitch + t0 + (lane >> 2);
#pragma unroll
      for (uint32_t n = 0; n < 4; ++n)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
          if (!open) {
            const int32_t q = s.query[8 * (nt0 + n) + 2 * (lane & 3) + (e & 1)];
            const uint32_t key = e >> 1 ? kb : ka;
            if (q < 0 || key > (uint32_t)q || key < window_start((uint32_t)q, a.window)) x[n][e] = INT32_MIN;
          }
          __stcg(out + (8 * n + (e & 1)) * sc.pitch + 8 * (e >> 1), x[n][e]);
        }
#pragma unroll
      for (uint32_t n = 0; n < 4; ++n)
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) {
          int32_t m = max(x[n][e], x[n][e + 2]);
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
          if (lane < 4) atomicMax(&s.top[8 * (nt0 + n) + 2 * lane + e], m);
        }
    }
    __syncthreads();

    // 2. terms in place, sums, first maxima. Where a row's maximum is within
    // 16.0 of the lowest score that mark does not tell hidden keys, and the
    // causal range is asked again.
    const uint32_t written = (p.count + 15) / 16 * 16, padded = (p.count + 31) / 32 * 32;
    int4 x[2];  // a row's first scores, loaded during the row before
    row_load(x, scores + (uint64_t)warp * sc.pitch, 128, 0, written, lane);
    for (uint32_t i = warp; i < RT; i += kPromptWarps) {
      const int32_t top = s.top[i], q = s.query[i];
      int32_t* row = scores + (uint64_t)i * sc.pitch;
      const int32_t* next = i + kPromptWarps < RT ? row + (uint64_t)kPromptWarps * sc.pitch : nullptr;
      uint64_t sum = 0;
      uint32_t first = UINT32_MAX;
      if (q >= 0 && top >= INT32_MIN + (1 << 20)) {
        const RowTerms r = row_terms(row, 128, written, padded, top, lists + warp * kTermList, lane, x, next);
        sum = r.sum;
        first = r.first;
      } else if (next) {
        row_load(x, next, 128, 0, written, lane);
      }
      if (q >= 0 && top < INT32_MIN + (1 << 20)) {
        for (uint32_t t = lane; t < padded; t += 32) {
          const uint32_t key = p.base + t;
          const bool gone = t >= p.count || key > (uint32_t)q || key < window_start((uint32_t)q, a.window);
          const uint32_t e = gone ? 0 : term_of(__ldcg(row + t), top);
          if (e == kTermTop) first = min(first, t);
          sum += kept_term(e);
          __stcg((uint32_t*)row + t, e);
        }
      }
      sum = (uint64_t)warp_sum_i64((int64_t)sum);
      first = __reduce_min_sync(0xffffffffu, first);
      __syncwarp();
      if (lane == 0) {
        s.sum[i] = sum;
        s.first[i] = first;
        if (q >= 0) __stcg(row + first, 0);  // its weight comes last
      }
    }
    __syncwarp();
    if (lane < RT / kPromptWarps) s.recip[warp + lane * kPromptWarps] = sum_recip(s.sum[warp + lane * kPromptWarps]);
    __syncthreads();

    // 3. weights and value sums
    if (prompt_values<RT, 3>(a, p, s, w, scores, sc.pitch, acc_buf))
      prompt_values<RT, 4>(a, p, s, w, scores, sc.pitch, acc_buf);
  }
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Rows of a tile: 64, or 32 for heads past 128 values (a warp's value sums
// cover 16 dimensions x 32 rows, sixteen warps).
uint32_t row_tile(const IrisPromptAttention& a) { return a.head_dim <= 128 ? 64 : 32; }

// The tensor-core kernel's packing and its two further launches pay for one
// long request, whose tiles wait for their longest, or where there is much to
// multiply. Measured, us, there against here: 32 query heads, 8 K/V heads of 128:
// 384 rows 81 / 70, 512 rows 93 / 101, 1,024 rows 195 / 298, thirty-two requests of
// 130 455 / 507; 8 heads and 1 of 256: 512 rows 81 / 61, 1,024 rows 115 / 120, four
// requests of 256 68 / 65, of 512 128 / 152; 4 heads and 1 of 64: 512 rows 65 / 60,
// 1,024 rows 89 / 104, sixteen requests of 256 85 / 75.
bool on_tensor_cores(const IrisPromptAttention& a) {
  const uint64_t pairs = (uint64_t)a.tokens * a.longest;
  return (a.longest >= 1024 || (a.longest >= 128 && pairs / 1024 * a.heads * a.head_dim >= 1u << 20)) &&
         prompt_tc_usable(a);
}

size_t carve(const IrisPromptAttention& a, uint8_t* base, PromptScratch* sc, PromptTcScratch* tc) {
  const uint32_t rt = row_tile(a), group = a.heads / a.kv_heads, most = on_tensor_cores(a) ? 64 : rt;
  const uint64_t tiles = ((uint64_t)a.tokens * group + rt - 1) / rt + a.requests;
  sc->blocks = (uint32_t)std::min<uint64_t>(tiles * a.kv_heads, (uint64_t)device_sms());
  const uint64_t keys = a.window ? std::min<uint64_t>(a.longest, (uint64_t)a.window + most + 16) : a.longest;
  sc->pitch = (uint32_t)((keys + 15 + 127) / 128 * 128);  // a tile's first key is rounded down to 16, its last up to 128
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = base + at;
    at += up256(bytes);
    return p;
  };
  // a tile a block: nothing to balance, and no launch for the list
  if (!on_tensor_cores(a) && a.requests <= kFewRequests && tiles * a.kv_heads <= (uint64_t)device_sms()) {
    sc->next = sc->order = sc->tiles = nullptr;
    sc->scores = (int32_t*)take((size_t)sc->blocks * rt * sc->pitch * 4);
    sc->acc = (int64_t*)take((size_t)sc->blocks * rt * a.head_dim * 8);
    sc->wide = nullptr;
    sc->flags = 0;
    return at;
  }
  sc->next = (uint32_t*)take(8);
  sc->tiles = (uint32_t*)take(((size_t)a.requests + 1) * 4);
  sc->tc_tiles = (uint32_t*)take(((size_t)a.requests + 1) * 4);
  sc->order = (uint32_t*)take((size_t)a.requests * 4);
  sc->scores = (int32_t*)take((size_t)sc->blocks * most * sc->pitch * 4);
  sc->acc = (int64_t*)take((size_t)sc->blocks * rt * a.head_dim * 8);
  sc->wide = nullptr;
  sc->flags = 0;
  if (on_tensor_cores(a)) {
    at += prompt_tc_carve(a, base + at, tc);
    tc->order = sc->order;
    tc->tiles = sc->tc_tiles;
    tc->next = sc->next + 1;
    tc->scores = sc->scores;
    tc->pitch = sc->pitch;
    sc->wide = tc->wide;
    sc->flags = tc->flags;
  }
  return at;
}

template <uint32_t RT>
cudaError_t launch(const IrisPromptAttention& a, const PromptScratch& sc, const PromptTcScratch& tc,
                   cudaStream_t stream) {
  const uint32_t smem = RT / 8 * (a.head_dim / 32) * 1024 + 2 * kPromptKeys / 32 * (RT / 8) * 512 +
                        kPromptWarps * kTermList * 4;
  static std::atomic<bool> allowed[64];
  cudaError_t e = allow_smem(prompt_mma_kernel<RT>, allowed);
  if (e != cudaSuccess) return e;
  if (!sc.order) {
    prompt_mma_kernel<RT><<<sc.blocks, kPromptThreads, smem, stream>>>(a, sc);
    return cudaGetLastError();
  }
  prompt_items_kernel<<<sc.flags ? 2 : 1, 1024, 0, stream>>>(a, sc, RT);
  e = cudaGetLastError();
  if (e == cudaSuccess && sc.flags) e = launch_prompt_tc(a, tc, sc.blocks, stream);
  if (e != cudaSuccess) return e;
  return launch_k(prompt_mma_kernel<RT>, dim3(sc.blocks), dim3(kPromptThreads), smem, stream, a, sc);
}

}  // namespace

bool prompt_mma_usable(const IrisPromptAttention& a) {
  return a.head_dim % 32 == 0 && a.scale_q32 < 0x80000000u && (uint64_t)a.tokens * a.heads < 0x80000000ull;
}

uint64_t prompt_mma_workspace(const IrisPromptAttention& a) {
  PromptScratch sc;
  PromptTcScratch tc;
  return carve(a, nullptr, &sc, &tc);
}

cudaError_t launch_prompt_mma(const IrisPromptAttention& a, uint8_t* workspace, cudaStream_t stream) {
  PromptScratch sc;
  PromptTcScratch tc;
  carve(a, workspace, &sc, &tc);
  return row_tile(a) == 64 ? launch<64>(a, sc, tc, stream) : launch<32>(a, sc, tc, stream);
}

}  // namespace iris
