// Drafted trees on the tcgen05 tensor cores (kind::i8), head_dim up to 128
// (narrower heads padded with zeros in shared memory): the first and third
// launches of tree_mma.cu with their contractions on the fifth-generation tensor
// cores.
//
// Keys and values are read where they lie in their pages, once: sixteen warps
// turn 128 of them into swizzled planes of signed base-256 digits in shared
// memory (24-bit values, nearly; a wider one is flagged and the launches of
// tree_mma.cu behind these do the work), while the products of the tile before
// run. Scores: a key plane against the three planes of 64 query rows side by side
// (128 x 192 x 32 a product) into five int32 diagonals in TMEM, all row tiles of a
// head against a tile of keys before the next. Values: a transposed value plane
// against both weight planes of 64 or 128 rows into four diagonals that stay in
// TMEM over the block's keys. A seventeenth warp issues the products (a warp that
// also worked on the scores held the others up: 777 against 732 us in all); every
// wait is bounded and a give-up ends the block and is recorded in the fault word.
//
// 64 and 48 nodes over 32,001 and 20,011 keys (32 query heads, 8 of 128 values): 251
// us for the scores, 248 us for the values, of 700. The products' unit is busy a
// tenth of the time, and the scores leave half of the issue slots empty (integer
// pipes 41 % busy): bound by the latency of a block's one chain of loading and
// splitting keys, waiting for products and finishing scores, with one block a
// multiprocessor (without the score's stores, the maxima, or three quarters of the
// products they take 1 to 5 % less); the values by the reading of the terms (the
// scratch is 384 MB there) and the weights' arithmetic. A value past 24 bits that
// the call names runs the launches of tree_mma.cu after these: 1,330 to 1,460 us in
// all, and 513 to 527 for the trees of a batch that take 245.
#include <algorithm>

#include "../../include/iris_b200.h"
#include "common.cuh"
#include "q8.cuh"
#include "serve_tc.cuh"
#include "tree_tc.cuh"

namespace iris {

namespace {

constexpr uint32_t kTtD = 128, kTtKeys = 128, kTtWarps = 16, kTtWork = 32 * kTtWarps;
constexpr uint32_t kTtThreads = kTtWork + 32;         // and one warp that issues the products
constexpr uint32_t kTtTile = 64;                      // query rows of a score tile
constexpr uint32_t kTtRows = kTreeTcRows;             // query rows a scores block holds
constexpr uint32_t kTtPlane = kTtKeys * kTtD;         // bytes of a key or value plane
constexpr uint32_t kTtQPlane = kTtTile * kTtD;

__device__ __forceinline__ uint8_t* aligned_1024(uint8_t* p) {
  return (uint8_t*)(((uintptr_t)p + 1023) & ~(uintptr_t)1023);
}

struct TtBlock {  // TMEM and its waits
  uint64_t drained;
  uint32_t tmem, dead, wide;
};

__device__ __forceinline__ void tt_alloc(TtBlock& s, uint32_t warp, uint32_t cols) {
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s.tmem)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
// The last warp issued the products.
__device__ __forceinline__ void tt_free(TtBlock& s, uint32_t warp, uint32_t cols, unsigned int* fault) {
  if (warp == kTtWarps && s.dead) tc_drain(&s.drained, (threadIdx.x & 31) == 0, fault);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem), "r"(cols) : "memory");
  }
}

// ---- scores ---------------------------------------------------------------------

struct TtScores {
  TtBlock b;
  uint64_t ready;             // a score tile's products are done
  uint64_t taken;             // and out of TMEM, the next tile's keys in shared memory
  uint64_t row_at[kTtRows];   // the rows' scores
  uint64_t mask[kTtRows];     // the nodes a row sees
  uint32_t position[kTtRows];
  int32_t top[kTtRows];
};

__global__ void __launch_bounds__(kTtThreads, 1)
    tree_tc_scores_kernel(IrisTreeAttention a, TreeScratch sc, uint32_t row_groups, unsigned int* fault) {
  extern __shared__ uint8_t tt_raw[];
  __shared__ __align__(16) TtScores s;
  uint8_t* keys = aligned_1024(tt_raw);   // two tiles of three planes
  uint8_t* qs = keys + 2 * 3 * kTtPlane;  // three planes a row tile
  const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t chunk = blockIdx.x, g = blockIdx.y / row_groups, r = blockIdx.z;
  const uint32_t f0 = blockIdx.y % row_groups * kTtRows;
  const TreeRequest q(a, r);
  const uint32_t rows_all = q.nodes * q.group, key0 = q.base + chunk * sc.chunk;
  if (key0 >= q.keys || f0 >= rows_all) return;
  const uint32_t rows = min(kTtRows, rows_all - f0), rts = (rows + kTtTile - 1) / kTtTile;
  const uint32_t count = min(sc.chunk, q.keys - key0), kts = (count + kTtKeys - 1) / kTtKeys;
  const int32_t* table = a.table + (size_t)r * a.width;
  const size_t kvd = (size_t)a.kv_heads * a.head_dim;
  const uint32_t stand_in = stand_in_row(a, q, table);
  const bool used = 4 * lane < a.head_dim;  // the lane's four dims
  const int4 none = make_int4(0, 0, 0, 0);

  if (tid == 0) {
    mbar_init(&s.ready, 1);
    mbar_init(&s.taken, kTtWarps);
    mbar_init(&s.b.drained, 1);
    s.b.dead = 0;
    s.b.wide = 0;
    mbar_fence_init();
  }
  tt_alloc(s.b, warp, 512);
  for (uint32_t i = tid; i < rts * kTtTile; i += kTtThreads) {  // (rows past the last one repeat it)
    const uint32_t f = f0 + min(i, rows - 1), node = q.node_of(f), head = q.head_of(f, g);
    const uint32_t row = q.begin + node;
    s.row_at[i] = ((size_t)row * a.heads + head) * sc.pitch;
    s.mask[i] = (uint64_t)a.masks[row] & node_bits(q.nodes);
    s.position[i] = a.positions ? (uint32_t)a.positions[row] : 0;
    s.top[i] = INT32_MIN;
  }
  uint32_t wide = 0;
  const bool works = warp < kTtWarps;  // (the last warp issues)
  // the query rows: a warp a row and turn, four values a lane
  if (works) {
#pragma unroll 1
    for (uint32_t i0 = warp; i0 < rts * kTtTile; i0 += 4 * kTtWarps) {
      int4 x[4];
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t f = f0 + min(i0 + u * kTtWarps, rows - 1);
        const int32_t* src = a.q + (size_t)(q.begin + q.node_of(f)) * a.q_stride + q.head_of(f, g) * a.head_dim;
        x[u] = used ? *(const int4*)(src + 4 * lane) : none;
      }
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t i = i0 + u * kTtWarps;  // (a row tile is four turns of the warps)
        uint32_t p[4];
        split_digits(x[u].x, x[u].y, x[u].z, x[u].w, p);
        wide |= p[3];
        uint8_t* dst = qs + i / kTtTile * 3 * kTtQPlane + swizzled(i % kTtTile, 4 * lane);
#pragma unroll
        for (uint32_t j = 0; j < 3; ++j) *(uint32_t*)(dst + j * kTtQPlane) = p[j];
      }
    }
  }
  // the keys of a tile: a warp takes eight of them, four values a lane
  int4 x[8];
  // (the table's entries are read a tile ahead of the keys)
  const uint32_t quad = warp & 3, cg = warp >> 2, tiles = kts * rts;
  auto table_at = [&](uint32_t t) {
    const uint32_t column = (key0 + t) / a.page_size;
    return t < count && column < a.width ? table[column] : -1;
  };
  int32_t id_key = -1, id_score = -1;  // of the lane's key to load, and of the key of its scores
  auto look_up = [&](uint32_t kt) {
    if (kt >= kts) return;
    id_key = table_at(kt * kTtKeys + warp * 8 + (lane & 7));
    id_score = table_at(kt * kTtKeys + 32 * quad + lane);
  };
  auto load_keys = [&](uint32_t kt) {
    const uint32_t at = key0 + kt * kTtKeys + warp * 8 + (lane & 7);
    const int64_t row = id_key < 0 || (uint64_t)id_key >= a.pages ? stand_in : (int64_t)id_key * a.page_size + at % a.page_size;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const int32_t* src = a.k_pages + (size_t)__shfl_sync(0xffffffffu, row, i) * kvd + g * a.head_dim;
      x[i] = used ? *(const int4*)(src + 4 * lane) : none;
    }
  };
  auto put_keys = [&](uint32_t kt) {
    uint8_t* dst = keys + (kt & 1) * 3 * kTtPlane;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      uint32_t p[4];
      split_digits(x[i].x, x[i].y, x[i].z, x[i].w, p);
      wide |= p[3];
      const uint32_t at = swizzled(warp * 8 + i, 4 * lane);
#pragma unroll
      for (uint32_t j = 0; j < 3; ++j) *(uint32_t*)(dst + j * kTtPlane + at) = p[j];
    }
  };
  // whether the key of a lane's scores is there, its page in the pool
  auto in_pool = [&] { return id_score >= 0 && (uint64_t)id_score < a.pages; };
  bool there = false, there_next = false;
  if (works) {
    look_up(0);
    load_keys(0);
    there = in_pool();
    look_up(1);
    put_keys(0);
    if (kts > 1) {
      load_keys(1);
      there_next = in_pool();
      look_up(2);
    }
  }
  fence_async_shared();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.b.tmem;
  if (!works) {
    // one score tile's products: plane i of the keys against all three of the
    // rows is diagonals i, i + 1, i + 2; a diagonal's first product overwrites it
    const uint64_t keys_d = tc_desc(smem_addr(keys)), qs_d = tc_desc(smem_addr(qs));
    const bool leader = lane == 0;
    for (uint32_t n = 0; n < tiles; ++n) {
      if (n && !tc_wait(&s.taken, (n - 1) & 1, &s.b.dead, fault)) break;
      __syncwarp();
      tc_fence_after();
      const uint32_t kt = n / rts, rt = n % rts;
      const uint64_t kd = keys_d + (kt & 1) * (3 * kTtPlane / 16), qd = qs_d + rt * (3 * kTtQPlane / 16);
#pragma unroll
      for (uint32_t i = 0; i < 3; ++i) {
        const uint64_t key = kd + i * (kTtPlane / 16);
        const uint32_t col = tmem + i * kTtTile;
        if (i == 0) {
          tc_mma_by(col, key, qd, tc_idesc_n(true, true, 3 * kTtTile), false, leader);
        } else {
          tc_mma_by(col, key, qd, tc_idesc_n(true, true, 2 * kTtTile), true, leader);
          tc_mma_by(col + 2 * kTtTile, key, qd + 2 * (kTtQPlane / 16), tc_idesc_n(true, true, kTtTile), false, leader);
        }
#pragma unroll
        for (uint32_t kk = 1; kk < 4; ++kk)
          tc_mma_by(col, key + 2 * kk, qd + 2 * kk, tc_idesc_n(true, true, 3 * kTtTile), true, leader);
      }
      tc_commit_by(&s.ready, leader);
    }
  } else {
    for (uint32_t n = 0; n < tiles; ++n) {
      const uint32_t kt = n / rts, rt = n % rts;
      // With a key tile's last row tile the next keys, loaded one tile ahead, go
      // to the other buffer (its products were waited for before).
      const bool turn = rt + 1 == rts;
      if (turn && kt + 1 < kts) {
        put_keys(kt + 1);
        fence_async_shared();
      }
      if (!tc_wait(&s.ready, n & 1, &s.b.dead, fault)) break;
      __syncwarp();
      tc_fence_after();
      uint32_t lo[16];
      int32_t hi[16];
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        uint32_t v[5][8];
#pragma unroll
        for (uint32_t d = 0; d < 5; ++d) tmem_ld8(tmem + ((32 * quad) << 16) + d * kTtTile + cg * 16 + h * 8, v[d]);
        tmem_ld_wait();
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c) {
          const int32_t w[5] = {(int32_t)v[0][c], (int32_t)v[1][c], (int32_t)v[2][c], (int32_t)v[3][c], (int32_t)v[4][c]};
          sum_digits<kTtD>(w, &hi[h * 8 + c], &lo[h * 8 + c]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.taken);
      int32_t y[16];
      scores_of(hi, lo, a.scale_q32, y);
      const uint32_t k = kt * kTtKeys + 32 * quad + lane, key = key0 + k;
      if (a.window || !__all_sync(0xffffffffu, there && key < q.held)) {
        // a node's key: its bit in the rows' masks, and its position
        const uint32_t node = key - q.held;
        const uint64_t bit = key < q.held ? ~0ull : node < kTreeNodes ? 1ull << node : 0;
        const uint32_t at = key < q.held ? key : a.window && there ? (uint32_t)a.positions[q.begin + node] : 0;
#pragma unroll
        for (uint32_t c = 0; c < 16; ++c) {
          const uint32_t i = rt * kTtTile + cg * 16 + c;
          if (!there || !(key < q.held || (s.mask[i] & bit)) || (a.window && at + a.window <= s.position[i])) y[c] = INT32_MIN;
        }
      }
      int32_t* out = sc.scores + (key - q.base);
      if (key - q.base < sc.pitch) {
#pragma unroll
        for (uint32_t c = 0; c < 16; ++c) out[s.row_at[rt * kTtTile + cg * 16 + c]] = y[c];
      }
      __syncwarp();
      int32_t best = INT32_MIN;
#pragma unroll
      for (uint32_t c = 0; c < 16; ++c) {
        const int32_t m = __reduce_max_sync(0xffffffffu, y[c]);
        best = lane == c ? m : best;
      }
      if (lane < 16) atomicMax(&s.top[rt * kTtTile + cg * 16 + lane], best);
      if (turn) {
        there = there_next;
        if (kt + 2 < kts) {
          load_keys(kt + 2);
          there_next = in_pool();
          look_up(kt + 3);
        }
      }
    }
  }
  if (wide) s.b.wide = 1;
  __syncthreads();
  for (uint32_t i = tid; i < rows; i += kTtThreads) sc.chunk_max[s.row_at[i] / sc.pitch * sc.chunks + chunk] = s.top[i];
  if (tid == 0 && s.b.wide) atomicOr(sc.flags, 1u);
  tt_free(s.b, warp, 512, fault);
}

// ---- values -----------------------------------------------------------------------

template <uint32_t RB>
struct TtValues {
  TtBlock b;
  uint64_t done[2];  // the products of a stage's buffers
  uint64_t full[2];  // a stage's values and weights are in shared memory
  uint64_t sum[RB];
  uint32_t recip[RB], first[RB], id[RB];  // id: the row's place in the scratch, UINT32_MAX past the last
  uint32_t last;
};

// RB rows of one request and K/V head, a chunk of its keys in stages of 128.
template <uint32_t RB>
__global__ void __launch_bounds__(kTtThreads, 1)
    tree_tc_values_kernel(IrisTreeAttention a, TreeScratch sc, unsigned int* fault) {
  constexpr uint32_t kWPlane = RB * kTtKeys, kUnits = RB * 16 / kTtWork;  // a thread's units of eight weights
  extern __shared__ uint8_t tt_raw[];
  __shared__ __align__(16) TtValues<RB> s;
  uint8_t* vals = aligned_1024(tt_raw);                       // two stages of three planes [dim][128 keys]
  uint8_t* wts = vals + 2 * 3 * kTtPlane;                     // two stages of two planes [row][128 keys]
  uint32_t* row_s = (uint32_t*)(wts + 2 * 2 * kWPlane);       // pool rows of the chunk's keys
  const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t chunk = blockIdx.x, g = blockIdx.y / sc.tc_groups, r = blockIdx.z;
  const uint32_t f0 = blockIdx.y % sc.tc_groups * RB;
  const TreeRequest q(a, r);
  const uint32_t rows = q.nodes * q.group, s0 = chunk * sc.tc_vchunk, key0 = q.base + s0;
  const uint32_t chunks = (q.count + sc.tc_vchunk - 1) / sc.tc_vchunk, segs = (q.count + kTreeSegment - 1) / kTreeSegment;
  if (f0 >= rows || key0 >= q.keys) return;
  const uint32_t count = min(sc.tc_vchunk, (q.keys - key0 + 31) / 32 * 32), stages = (count + kTtKeys - 1) / kTtKeys;
  const int32_t* table = a.table + (size_t)r * a.width;
  const size_t kvd = (size_t)a.kv_heads * a.head_dim;
  const uint32_t stand_in = stand_in_row(a, q, table);
  for (uint32_t i = tid; i < stages * kTtKeys; i += kTtThreads) {
    const int64_t row = key0 + i < q.keys ? page_row(table, a.width, a.page_size, a.pages, key0 + i) : -1;
    row_s[i] = row < 0 ? stand_in : (uint32_t)row;
  }
  if (tid == 0) {
    mbar_init(&s.done[0], 1);
    mbar_init(&s.done[1], 1);
    mbar_init(&s.full[0], kTtWarps);
    mbar_init(&s.full[1], kTtWarps);
    mbar_init(&s.b.drained, 1);
    s.b.dead = 0;
    s.b.wide = 0;
    mbar_fence_init();
  }
  tt_alloc(s.b, warp, 4 * RB);
  __syncthreads();
  // values: a warp's two units of 16 keys x 32 dims, a dim a lane
  const uint32_t dim = (warp & 3) * 32 + lane;
  int32_t x[2][16];
  auto load_values = [&](uint32_t st) {
    const int32_t* v = a.v_pages + g * a.head_dim + (dim < a.head_dim ? dim : 0);  // (dims past the head's are not stored)
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      const uint4* row = (const uint4*)(row_s + st * kTtKeys + ((warp >> 2) + 4 * u) * 16);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint4 k = row[j];
        x[u][4 * j] = v[(size_t)k.x * kvd];
        x[u][4 * j + 1] = v[(size_t)k.y * kvd];
        x[u][4 * j + 2] = v[(size_t)k.z * kvd];
        x[u][4 * j + 3] = v[(size_t)k.w * kvd];
      }
    }
  };
  const bool works = warp < kTtWarps;  // (the last warp issues)
  if (works) load_values(0);
  pdl_wait();
#pragma unroll 4
  for (uint32_t i = warp; works && i < RB; i += kTtWarps) {
    const uint32_t f = f0 + i;
    uint64_t sum = 0;
    uint32_t first = UINT32_MAX, id = UINT32_MAX;
    if (f < rows) {
      id = (q.begin + q.node_of(f)) * a.heads + q.head_of(f, g);
      for (uint32_t y = lane; y < segs; y += 32) {
        sum += sc.seg_sum[(size_t)id * sc.segs + y];
        first = min(first, sc.seg_first[(size_t)id * sc.segs + y]);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.b.tmem;
  uint4 t[kUnits][2];
  // unit u of a thread: eight keys of row tid / 16 + 32 u
  auto load_terms = [&](uint32_t st) {
#pragma unroll
    for (uint32_t u = 0; u < kUnits; ++u) {
      const uint32_t id = s.id[(tid >> 4) + 32 * u], at = st * kTtKeys + 8 * (tid & 15);
      t[u][0] = t[u][1] = make_uint4(0, 0, 0, 0);
      if (id != UINT32_MAX && at < count) {
        const int32_t* e = sc.scores + (size_t)id * sc.pitch + s0 + at;
        t[u][0] = __ldcg((const uint4*)e);
        t[u][1] = __ldcg((const uint4*)(e + 4));
      }
    }
  };
  if (works) load_terms(0);
  uint32_t wide = 0;
  int32_t total[kUnits] = {};
  bool ok = true;
  if (!works) {
    // value plane i against both weight planes: diagonals i, i + 1
    const uint64_t vals_d = tc_desc(smem_addr(vals)), wts_d = tc_desc(smem_addr(wts));
    const bool leader = lane == 0;
    for (uint32_t st = 0; st < stages; ++st) {
      const uint32_t buf = st & 1;
      if (!tc_wait(&s.full[buf], (st >> 1) & 1, &s.b.dead, fault)) break;
      __syncwarp();
      tc_fence_after();
      const uint64_t vd = vals_d + buf * (3 * kTtPlane / 16), wd = wts_d + buf * (2 * kWPlane / 16);
#pragma unroll
      for (uint32_t i = 0; i < 3; ++i) {
        const uint64_t val = vd + i * (kTtPlane / 16);
        const uint32_t col = tmem + i * RB;
        if (st == 0 && i) {
          tc_mma_by(col, val, wd, tc_idesc_n(true, false, RB), true, leader);
          tc_mma_by(col + RB, val, wd + kWPlane / 16, tc_idesc_n(true, false, RB), false, leader);
        } else {
          tc_mma_by(col, val, wd, tc_idesc_n(true, false, 2 * RB), st != 0, leader);
        }
#pragma unroll
        for (uint32_t kk = 1; kk < 4; ++kk)
          tc_mma_by(col, val + 2 * kk, wd + 2 * kk, tc_idesc_n(true, false, 2 * RB), true, leader);
      }
      tc_commit_by(&s.done[buf], leader);
    }
  }
  for (uint32_t st = 0; works && st < stages; ++st) {
    const uint32_t buf = st & 1;
    if (st >= 2) {
      ok = tc_wait(&s.done[buf], ((st >> 1) - 1) & 1, &s.b.dead, fault);
      if (!ok) break;
      __syncwarp();
    }
    uint8_t* vb = vals + buf * 3 * kTtPlane;
    uint8_t* wb = wts + buf * 2 * kWPlane;
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      uint32_t p[4][4];  // [four keys][plane]
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        split_digits(x[u][4 * j], x[u][4 * j + 1], x[u][4 * j + 2], x[u][4 * j + 3], p[j]);
        wide |= p[j][3];
      }
      const uint32_t at = swizzled(dim, 16 * ((warp >> 2) + 4 * u));
#pragma unroll
      for (uint32_t i = 0; i < 3; ++i)
        *(uint4*)(vb + i * kTtPlane + at) = make_uint4(p[0][i], p[1][i], p[2][i], p[3][i]);
    }
#pragma unroll
    for (uint32_t u = 0; u < kUnits; ++u) {
      const uint32_t i = (tid >> 4) + 32 * u, c = tid & 15;
      const uint32_t e[8] = {t[u][0].x, t[u][0].y, t[u][0].z, t[u][0].w, t[u][1].x, t[u][1].y, t[u][1].z, t[u][1].w};
      int32_t w[8];
      weights_of(e, s.recip[i], s.sum[i], w);
      const uint32_t first = s.first[i] - (s0 + st * kTtKeys + 8 * c);
      if (first < 8) {  // its weight comes last
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) w[j] = j == first ? 0 : w[j];
      }
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) total[u] += w[j];
      const uint32_t t0 = __byte_perm(w[0], w[1], 0x5140), t1 = __byte_perm(w[2], w[3], 0x5140);
      const uint32_t u0 = __byte_perm(w[4], w[5], 0x5140), u1 = __byte_perm(w[6], w[7], 0x5140);
      uint8_t* dst = wb + swizzled(i, 8 * c);
      *(uint2*)dst = make_uint2(__byte_perm(t0, t1, 0x5410), __byte_perm(u0, u1, 0x5410));
      *(uint2*)(dst + kWPlane) = make_uint2(__byte_perm(t0, t1, 0x7632), __byte_perm(u0, u1, 0x7632));
    }
    fence_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.full[buf]);
    if (st + 1 < stages) {
      load_values(st + 1);
      load_terms(st + 1);
    }
  }
  if (wide) s.b.wide = 1;
  // every stage's products before the totals are read (the last commit covers all)
  if (ok) ok = tc_wait(&s.done[(stages - 1) & 1], ((stages - 1) >> 1) & 1, &s.b.dead, fault);
  tc_fence_after();
  const uint32_t quad = warp & 3, cg = warp >> 2;
  if (ok && works) {
#pragma unroll 1
    for (uint32_t c0 = 0; c0 < RB / 4; c0 += 8) {
      uint32_t v[4][8];
#pragma unroll
      for (uint32_t d = 0; d < 4; ++d) tmem_ld8(tmem + ((32 * quad) << 16) + d * RB + cg * (RB / 4) + c0, v[d]);
      tmem_ld_wait();
#pragma unroll
      for (uint32_t c = 0; c < 8; ++c) {
        const uint32_t id = s.id[cg * (RB / 4) + c0 + c];
        const int32_t y[4] = {(int32_t)v[0][c], (int32_t)v[1][c], (int32_t)v[2][c], (int32_t)v[3][c]};
        if (id != UINT32_MAX && 32 * quad + lane < a.head_dim)
          atomicAdd((unsigned long long*)(sc.tc_acc + (size_t)id * a.head_dim + 32 * quad + lane),
                    (unsigned long long)diagonal_sum(y));
      }
    }
  }
#pragma unroll
  for (uint32_t u = 0; works && u < kUnits; ++u) {
    int32_t y = total[u];
#pragma unroll
    for (uint32_t o = 1; o <= 8; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    const uint32_t id = s.id[(tid >> 4) + 32 * u];
    if ((lane & 15) == 0 && id != UINT32_MAX && y) atomicAdd(sc.tc_wsum + id, y);
  }
  __syncthreads();
  // the last block of these rows writes the outputs
  if (tid == 0) {
    if (s.b.wide) atomicOr(sc.flags + 1, 1u);
    __threadfence();
    s.last = atom_add_acq_rel(sc.tc_done + ((size_t)r * a.kv_heads + g) * sc.tc_groups + f0 / RB, 1u) + 1 == chunks;
    __threadfence();
  }
  __syncthreads();
  if (s.last) {
    for (uint32_t i = warp; i < min(RB, rows - f0); i += kTtThreads / 32) {
      const uint32_t node = q.node_of(f0 + i), head = q.head_of(f0 + i, g), first = s.first[i];
      const size_t id = s.id[i];
      const int64_t row = first < q.count ? page_row(table, a.width, a.page_size, a.pages, q.base + first) : -1;
      const int32_t top = sub_sat(kOneAct, __ldcg(sc.tc_wsum + id));
      int32_t* out = a.out + (size_t)(q.begin + node) * a.out_stride + head * a.head_dim;
      for (uint32_t y = lane; y < a.head_dim; y += 32) {
        int64_t sum = __ldcg(sc.tc_acc + id * a.head_dim + y);
        if (row >= 0) mac_wide(sum, top, a.v_pages[(size_t)row * kvd + g * a.head_dim + y]);
        out[y] = row >= 0 ? requantize(sum) : 0;
      }
    }
  }
  tt_free(s.b, warp, 4 * RB, fault);
}

uint32_t scores_smem(uint32_t row_tiles) { return 1024 + 2 * 3 * kTtPlane + row_tiles * 3 * kTtQPlane; }
uint32_t values_smem(uint32_t rows, uint32_t vchunk) { return 1024 + 2 * 3 * kTtPlane + 2 * 2 * rows * kTtKeys + vchunk * 4; }

template <uint32_t RB>
cudaError_t launch_values(const IrisTreeAttention& a, const TreeScratch& sc, cudaStream_t stream) {
  static std::atomic<bool> allowed[64];
  const cudaError_t e = allow_smem(tree_tc_values_kernel<RB>, allowed);
  if (e != cudaSuccess) return e;
  return launch_k(tree_tc_values_kernel<RB>, dim3(sc.tc_vchunks, a.kv_heads * sc.tc_groups, a.requests),
                  dim3(kTtThreads), values_smem(RB, sc.tc_vchunk), stream, a, sc, device_fault_word());
}

}  // namespace

// From 33 query rows of a K/V head on, 128 keys and more; for 17 to 32, which
// leave half of the 64-row products idle, only where much is to read. Measured, us,
// here against the mma.sync kernels (32 query heads, 8 K/V heads of 128): sixteen
// nodes over 256 keys 44.7 / 49.1, over 8,000 117 / 166; thirty-two nodes of sixteen
// requests over 8,000 1,101 / 1,962; eight nodes over 8,000 93 / 90, of sixteen
// requests over 777 128 / 122, over 2,000 196 / 201, over 8,000 542 / 616.
bool tree_tc_usable(const IrisTreeAttention& a) {
  const uint32_t rows = a.nodes * (a.heads / a.kv_heads);
  const uint64_t keys = (uint64_t)a.requests * a.kv_heads * a.longest;
  return a.head_dim <= kTtD && a.longest >= 128 && (rows > 32 || (rows > 16 && keys >= 1u << 18)) &&
         device_fault_word() != nullptr;
}

cudaError_t launch_tree_tc_scores(const IrisTreeAttention& a, const TreeScratch& sc, cudaStream_t stream) {
  static std::atomic<bool> allowed[64];
  const cudaError_t e = allow_smem(tree_tc_scores_kernel, allowed);
  if (e != cudaSuccess) return e;
  const uint32_t rows = a.nodes * (a.heads / a.kv_heads), groups = (rows + kTtRows - 1) / kTtRows;
  tree_tc_scores_kernel<<<dim3(sc.chunks, a.kv_heads * groups, a.requests), kTtThreads,
                          scores_smem((std::min(rows, kTtRows) + kTtTile - 1) / kTtTile), stream>>>(
      a, sc, groups, device_fault_word());
  return cudaGetLastError();
}

cudaError_t launch_tree_tc_values(const IrisTreeAttention& a, const TreeScratch& sc, cudaStream_t stream) {
  return sc.tc_rows == 64 ? launch_values<64>(a, sc, stream) : launch_values<128>(a, sc, stream);
}

}  // namespace iris
