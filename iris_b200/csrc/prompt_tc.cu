// Packed prompt attention on the tcgen05 tensor cores (kind::i8), heads of up to
// 256 values: in one or two chunks (DC) of 128, padded with zeros.
//
// The same three phases as prompt_mma.cu, with the contractions on the
// fifth-generation tensor cores. Operands are packed once a call into K-major
// byte planes (three signed digits: 24-bit values, nearly; where any operand is
// wider the kernel leaves the call to prompt_mma_kernel, launched behind it, which
// then runs):
// queries [K/V head][plane][token * group + head][128 DC], keys [head][plane]
// [token][128 DC], values transposed [head][plane][128 DC][token]. A tile of 64 query
// rows that share a K/V head goes through
//   1. scores: 128 keys x 192 rows x 32 dims a product (one key plane against
//      the three query planes side by side), nine plane pairs into five int32
//      diagonals of 64 TMEM columns; the epilogue warps carry the diagonals
//      together, release them and write the scores to the block's scratch (L2)
//      while the next tile's products run;
//   2. terms in place, a row a warp; an exponential is its polynomial in
//      double precision plus one bit of a table in shared memory that
//      makes it exact (exp_term_floor);
//   3. weights of 128 keys into shared memory as two swizzled byte planes, and
//      128 dims x 128 rows (both weight planes) x 32 positions a product, six
//      plane pairs into four diagonals that stay in TMEM over all keys.
// Products of 64 rows each took 148 cycles, whatever their order: the wide ones
// do three times the work in one.
// Sixteen epilogue warps, one warp that feeds the ring (16 KB, one plane of 128
// keys a slot) by TMA and one that issues the products. Every wait is bounded;
// a give-up ends the block and is recorded in the fault word.
//
// Requests of 4,096, 1,037, 711, 300 and 1 rows, 32 query heads over 8 of 128
// values: 1,897 us (295 M pairs, 79 TFLOP/s of the plain products); 1,025, 640, 512
// and 37 rows, 8 heads over one of 256: 134 us. Bound by the epilogue warps, not by
// the products (their unit is busy 12 %), and there by latency: half of the issue
// slots stay empty and the integer pipes are 37 % busy, since a block's sixteen warps
// take the three phases in strict turn and each waits for its loads of scores or
// terms (the largest stall). Of a tile's cycles 38 % are scores (2,800 for 128 keys
// x 64 rows: a 64-bit product and rounding each), 30 % the exact exponentials
// (3,300), 30 % weights and value sums, the wait for products a tenth of each. One
// value past 24 bits leaves the call to prompt_mma_kernel: 4,950 to 5,230 us and 264
// to 292 us for these two calls in all, against 1,960 and 150.
#include <algorithm>

#include "../../include/iris_b200.h"
#include "common.cuh"
#include "layers.cuh"
#include "prompt_tc.cuh"
#include "q8.cuh"
#include "serve_attn.cuh"
#include "serve_mma.cuh"
#include "serve_tc.cuh"
#include "tc.cuh"
#include "tcgen05.cuh"

namespace iris {

namespace {

constexpr uint32_t kPtD = 128, kPtRows = 64, kPtKeys = 128;  // dims of a chunk, query rows, keys of a tile
constexpr uint32_t kPtEpiWarps = 16, kPtEpi = 32 * kPtEpiWarps, kPtThreads = kPtEpi + 64;
constexpr uint32_t kPtSlot = kPtKeys * kPtD;     // one plane and chunk of a key or value tile
constexpr uint32_t kPtQPlane = kPtRows * kPtD;   // one plane and chunk of the query rows; of a weight tile
constexpr uint32_t kPtWBuf = 2 * kPtQPlane;      // two weight planes
constexpr uint32_t kPtBlock = kPtRows * kPtKeys;  // scores of a key tile: [row][key]
constexpr uint32_t kPtFar = kExpTerms - kExpExactBelow;  // distances with a correction bit
constexpr uint32_t kPtTable = kPtFar / 32;               // words
constexpr uint32_t kPtNearBits = 18;                     // kExpExactBelow below 2^18, places below 2^14
constexpr uint32_t kPtLongest = (1u << (32 - kPtNearBits)) - kPtKeys;
static_assert(kExpExactBelow < 1u << kPtNearBits, "list entries");
static_assert(kPtLongest + 15 + kPtKeys <= kPvKeys + kPtKeys, "int32 diagonals of the value sums");
static_assert(8 * kPtRows == 512, "TMEM column groups");

template <uint32_t DC>
struct PtLayout {
  static constexpr uint32_t kSlots = DC == 1 ? 5 : 3;
  static constexpr uint32_t kRing = kSlots * kPtSlot;
  static constexpr uint32_t kQuery = 3 * DC * kPtQPlane;  // [chunk][plane][row][128]
  static constexpr uint32_t kOperands = kQuery > 2 * kPtWBuf ? kQuery : 2 * kPtWBuf;  // the queries, later two weight buffers
  static constexpr uint32_t kList = kOperands / 4 / kPtEpiWarps;  // words of a warp's list of near scores
  static constexpr uint32_t kSmem = 1024 + kRing + kOperands + kPtTable * 4;
  static_assert(kList >= 512, "list entries");
};

// ---- packing -------------------------------------------------------------------

// Four values (zeros where src is NULL) into three planes; what is past 24 bits.
__device__ __forceinline__ uint32_t pack_row4(const int32_t* src, uint8_t* dst, uint64_t plane) {
  const int4 x = src ? *(const int4*)src : make_int4(0, 0, 0, 0);
  uint32_t p[4];
  split_digits(x.x, x.y, x.z, x.w, p);
#pragma unroll
  for (uint32_t i = 0; i < 3; ++i) *(uint32_t*)(dst + i * plane) = p[i];
  return p[3];
}

constexpr uint32_t kPackThreads = 256;

// blockIdx.y: 0 queries, 1 keys, 2 values (transposed through shared memory, 32
// tokens x 32 dims a pass), 3 the exponential's correction bits.
template <uint32_t DC>
__global__ void __launch_bounds__(kPackThreads) prompt_pack_kernel(IrisPromptAttention a, PromptTcScratch sc) {
  constexpr uint32_t DP = DC * kPtD;  // dims a packed row
  __shared__ int32_t tile[32][33];
  const uint32_t tid = threadIdx.x, group = a.heads / a.kv_heads;
  pdl_trigger();
  uint32_t wide = 0;
  if (blockIdx.y <= 1) {
    const bool keys = blockIdx.y == 1;
    const uint32_t per = keys ? 1 : group;
    const uint64_t rows = (uint64_t)a.tokens * per, n = rows * a.kv_heads * (DP / 4);
    const int32_t* src = keys ? a.k : a.q;
    const uint64_t stride = keys ? a.k_stride : a.q_stride;
    uint8_t* dst = keys ? sc.kp : sc.qp;
    for (uint64_t i = (uint64_t)blockIdx.x * kPackThreads + tid; i < n; i += (uint64_t)gridDim.x * kPackThreads) {
      const uint32_t c = (uint32_t)(i % (DP / 4)), h = (uint32_t)(i / (DP / 4) % (per * a.kv_heads));
      const uint64_t token = i / (DP / 4) / (per * a.kv_heads);
      const uint64_t row = token * per + h % per;
      wide |= pack_row4(4 * c < a.head_dim ? src + token * stride + (uint64_t)h * a.head_dim + 4 * c : nullptr,
                        dst + ((uint64_t)(h / per) * 3 * rows + row) * DP + 4 * c, rows * DP);
    }
  } else if (blockIdx.y == 2) {
    const uint32_t tx = tid & 31, ty = tid >> 5;
    const uint32_t tts = (a.tokens + 31) / 32;
    for (uint64_t u = blockIdx.x; u < (uint64_t)tts * (DP / 32) * a.kv_heads; u += gridDim.x) {
      const uint32_t g = (uint32_t)(u % a.kv_heads), d0 = (uint32_t)(u / a.kv_heads % (DP / 32)) * 32,
                     t0 = (uint32_t)(u / a.kv_heads / (DP / 32)) * 32;
      __syncthreads();
      for (uint32_t r = ty; r < 32; r += 8) {
        const uint32_t t = t0 + r;
        tile[r][tx] =
            t < a.tokens && d0 + tx < a.head_dim ? a.v[(uint64_t)t * a.v_stride + g * a.head_dim + d0 + tx] : 0;
      }
      __syncthreads();
      // thread: dimension tid / 8, four tokens
      const uint32_t d = tid >> 3, t = 4 * (tid & 7);
      uint32_t p[4];
      split_digits(tile[t][d], tile[t + 1][d], tile[t + 2][d], tile[t + 3][d], p);
      wide |= p[3];
#pragma unroll
      for (uint32_t i = 0; i < 3; ++i)
        *(uint32_t*)(sc.vt + (((uint64_t)g * 3 + i) * DP + d0 + d) * sc.tpitch + t0 + t) = p[i];
    }
  } else {
    const uint32_t lane = tid & 31;
    for (uint32_t c = blockIdx.x * kPackThreads + tid; c < kPtFar; c += gridDim.x * kPackThreads) {
      const uint32_t d = kExpExactBelow + c;
      const uint32_t bits = __ballot_sync(0xffffffffu, exp_term_near(d) != exp_term_floor(d));
      if (lane == 0) sc.exp_bits[c / 32] = bits;
    }
  }
  wide = __syncthreads_or(wide != 0);
  if (tid == 0) sc.wide[blockIdx.y * gridDim.x + blockIdx.x] = wide ? 1 : 0;
  pdl_wait();  // the item list, which the kernel after this one reads, is complete too
}

// ---- the attention ----------------------------------------------------------------

struct PtShared {
  uint64_t full[PtLayout<1>::kSlots], empty[PtLayout<1>::kSlots], q_full, s_done, t_free, w_full[2], w_empty[2], v_done, drained;
  uint64_t sum[kPtRows];
  int32_t top[kPtRows], query[kPtRows], wsum[kPtRows];
  uint32_t recip[kPtRows], first[kPtRows];
  uint32_t item, tmem, dead, wide;
};

__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kPtEpi) : "memory"); }
// The same barrier, and whether `x` holds for every epilogue warp.
__device__ __forceinline__ bool epi_all(bool x) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)x), "n"(kPtEpi)
      : "memory");
  return all != 0;
}

// The terms of eight scores, 0 below kExpExactBelow, and their distances.
__device__ __forceinline__ void terms_by_table(const int4 (&x)[2], int32_t top, const uint32_t* bits, uint32_t (&e)[8],
                                               uint32_t (&d)[8]) {
  const int32_t v[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
#pragma unroll
  for (uint32_t u = 0; u < 8; ++u) {
    d[u] = (uint32_t)top - (uint32_t)v[u];
    const uint32_t c = d[u] - kExpExactBelow, i = min(c, kPtFar - 1);
    const uint32_t t = exp_term_floor(d[u]) + (__funnelshift_r(bits[i >> 5], 0, i) & 1);
    e[u] = c < kPtFar ? t : 0;
  }
}

template <uint32_t DC>
__global__ void __launch_bounds__(kPtThreads, 1)
    prompt_tc_kernel(IrisPromptAttention a, PromptTcScratch sc, const __grid_constant__ CUtensorMap qmap,
                     const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     unsigned int* fault) {
  using L = PtLayout<DC>;
  constexpr uint32_t kPtSlots = L::kSlots, kPtList = L::kList;
  extern __shared__ uint8_t pt_raw[];
  __shared__ __align__(8) PtShared s;
  uint8_t* ring = (uint8_t*)(((uintptr_t)pt_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* ops = ring + L::kRing;  // query planes, then weight buffers
  uint32_t* bits = (uint32_t*)(ops + L::kOperands);
  const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const bool leader = lane == 0;
  if (tid == 0) {
    for (uint32_t i = 0; i < kPtSlots; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    mbar_init(&s.q_full, 1);
    mbar_init(&s.s_done, 1);
    mbar_init(&s.t_free, kPtEpiWarps);
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&s.w_full[i], kPtEpiWarps);
      mbar_init(&s.w_empty[i], 1);
    }
    mbar_init(&s.v_done, 1);
    mbar_init(&s.drained, 1);
    s.dead = 0;
    s.wide = 0;
    mbar_fence_init();
  }
  if (warp == kPtEpiWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s.tmem)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  pdl_wait();
  pdl_trigger();
  {
    uint32_t wide = 0;
    for (uint32_t i = tid; i < sc.flags; i += kPtThreads) wide |= sc.wide[i];
    if (wide) s.wide = 1;
    for (uint32_t i = tid; i < kPtTable; i += kPtThreads) bits[i] = sc.exp_bits[i];
  }
  __syncthreads();
  const bool run = s.wide == 0;
  const uint32_t items = run ? sc.tiles[a.requests] * a.kv_heads : 0, group = a.heads / a.kv_heads;
  int32_t* scores = sc.scores + (uint64_t)blockIdx.x * kPtRows * sc.pitch;
  const uint32_t ring_a = smem_addr(ring);
  const uint64_t ops_d = tc_desc(smem_addr(ops));

  // each role's running counts of the barriers' phases
  uint32_t ring_n = 0, n_item = 0, n_s = 0, n_w = 0;
  uint32_t issued[kPtSlots] = {};
  bool ok = true;
  for (;; ++n_item) {
    __syncthreads();  // the item before is done with the shared memory and the accumulators
    if (tid == 0) s.item = s.dead ? UINT32_MAX : atomicAdd(sc.next, 1u);
    __syncthreads();
    const uint32_t item = s.item;
    if (item >= items) break;
    const uint32_t g = item % a.kv_heads, at = item / a.kv_heads;
    const uint32_t rank = request_of(sc.tiles, a.requests, at), r = sc.order[rank];
    const uint32_t begin = clamp_offset(a.offsets[r], a.tokens);
    const uint32_t len = min(clamp_offset(a.offsets[r + 1], a.tokens) - begin, a.longest);
    const uint32_t f0 = (sc.tiles[rank + 1] - 1 - at) * kPtRows, rows = min(kPtRows, len * group - f0);
    const uint32_t q0 = f0 / group, q1 = (f0 + rows - 1) / group;
    // keys by their packed row from k0 on, a multiple of 16 (the transposed
    // values' TMA starts there); rows of other requests are hidden
    const uint32_t k0 = (begin + window_start(q0, a.window)) / 16 * 16, count = begin + q1 + 1 - k0;
    const uint32_t ktiles = (count + kPtKeys - 1) / kPtKeys;

    if (warp == kPtEpiWarps) {
      if (lane == 0) {  // TMA producer
        mbar_arrive_expect_tx(&s.q_full, L::kQuery);
        for (uint32_t j = 0; j < 3 * DC; ++j)
          tma_load_3d(ops + j * kPtQPlane, &qmap, (int32_t)(j / 3 * kPtD), (int32_t)(begin * group + f0),
                      (int32_t)(g * 3 + j % 3), &s.q_full);
        for (uint32_t u = 0; u < 6 * DC * ktiles && ok; ++u, ++ring_n) {
          const uint32_t slot = ring_n % kPtSlots, use = ring_n / kPtSlots;
          if (use > 0 && !tc_wait(&s.empty[slot], (use - 1) & 1, &s.dead, fault)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&s.full[slot], kPtSlot);
          const bool vals = u >= 3 * DC * ktiles;
          const uint32_t v = vals ? u - 3 * DC * ktiles : u, kt = v / (3 * DC), t = k0 + kt * kPtKeys;
          // a tile's planes, each in its chunks (every other score tile takes its planes from the last on)
          const uint32_t j = v / DC % 3, plane = g * 3 + (vals || ((n_s + kt) & 1) == 0 ? j : 2 - j);
          const int32_t c0 = (int32_t)(v % DC * kPtD);
          if (vals) tma_load_3d(ring + slot * kPtSlot, &vmap, (int32_t)t, c0, (int32_t)plane, &s.full[slot]);
          else tma_load_3d(ring + slot * kPtSlot, &kmap, c0, (int32_t)t, (int32_t)plane, &s.full[slot]);
          ++issued[slot];
        }
        n_s += ktiles;
      }
    } else if (warp == kPtEpiWarps + 1) {
      // product issuer: the whole warp walks the tiles (so that addresses and
      // descriptors stay uniform), its first lane issues
      ok = ok && tc_wait(&s.q_full, n_item & 1, &s.dead, fault);
      tc_fence_after();
      for (uint32_t kt = 0; kt < ktiles && ok; ++kt, ++n_s) {
        // Key plane i against the three query planes side by side (192 rows) is
        // diagonals i, i + 1, i + 2 in neighbouring column groups. The score
        // tiles take groups 0-4 and 3-7 in turn, from the end that the tile
        // before does not use, so a third of the products run while it is read.
        const bool up = (n_s & 1) == 0;
        const uint32_t cols = tmem + (up ? 0 : 3 * kPtRows);
#pragma unroll 1
        for (uint32_t u = 0; u < 3 * DC; ++u, ++ring_n) {
          const uint32_t st = u / DC, c = u % DC, i = up ? st : 2 - st, slot = ring_n % kPtSlots;
          ok = ok && tc_wait(&s.full[slot], (ring_n / kPtSlots) & 1, &s.dead, fault);
          if (u == DC && kt) ok = ok && tc_wait(&s.t_free, (n_s - 1) & 1, &s.dead, fault);
          if (!ok) break;
          tc_fence_after();
          const uint64_t key = tc_desc(ring_a + slot * kPtSlot), qd = ops_d + c * (3 * kPtQPlane / 16);
          const uint32_t col = cols + i * kPtRows;
          // the first product into a diagonal overwrites it: all three of the
          // first plane; then the outermost one of each further plane
          if (c == 0 && st == 0) {
            tc_mma_by(col, key, qd, tc_idesc_n(true, true, 3 * kPtRows), false, leader);
          } else if (c == 0) {
            const uint32_t in = up ? 0 : 1, out = up ? 2 : 0;  // query planes of the other two, and of the outermost
            tc_mma_by(col + in * kPtRows, key, qd + in * (kPtQPlane / 16), tc_idesc_n(true, true, 2 * kPtRows), true,
                      leader);
            tc_mma_by(col + out * kPtRows, key, qd + out * (kPtQPlane / 16), tc_idesc_n(true, true, kPtRows), false,
                      leader);
          } else {
            tc_mma_by(col, key, qd, tc_idesc_n(true, true, 3 * kPtRows), true, leader);
          }
#pragma unroll
          for (uint32_t kk = 1; kk < 4; ++kk)
            tc_mma_by(col, key + 2 * kk, qd + 2 * kk, tc_idesc_n(true, true, 3 * kPtRows), true, leader);
          tc_commit_by(&s.empty[slot], leader);
        }
        if (!ok) break;
        tc_commit_by(&s.s_done, leader);
      }
      // the diagonals of the last score tile are read before the value sums take their columns
      ok = ok && tc_wait(&s.t_free, (n_s - 1) & 1, &s.dead, fault);
      tc_fence_after();
      for (uint32_t kt = 0; kt < ktiles && ok; ++kt, ++n_w) {
        const uint32_t buf = n_w & 1;
        ok = tc_wait(&s.w_full[buf], (n_w >> 1) & 1, &s.dead, fault);
        // value plane i against both weight planes (128 rows): diagonals i, i + 1
        const uint64_t w = ops_d + buf * (kPtWBuf / 16);
#pragma unroll 1
        for (uint32_t u = 0; u < 3 * DC; ++u, ++ring_n) {
          // (dims 128 c .. have four column groups of their own)
          const uint32_t i = u / DC, c = u % DC, slot = ring_n % kPtSlots, col = tmem + (4 * c + i) * kPtRows;
          ok = ok && tc_wait(&s.full[slot], (ring_n / kPtSlots) & 1, &s.dead, fault);
          if (!ok) break;
          tc_fence_after();
          const uint64_t val = tc_desc(ring_a + slot * kPtSlot);
          if (kt == 0 && i) {
            tc_mma_by(col, val, w, tc_idesc_n(true, false, kPtRows), true, leader);
            tc_mma_by(col + kPtRows, val, w + kPtQPlane / 16, tc_idesc_n(true, false, kPtRows), false, leader);
          } else {
            tc_mma_by(col, val, w, tc_idesc_n(true, false, 2 * kPtRows), kt != 0, leader);
          }
#pragma unroll
          for (uint32_t kk = 1; kk < 4; ++kk)
            tc_mma_by(col, val + 2 * kk, w + 2 * kk, tc_idesc_n(true, false, 2 * kPtRows), true, leader);
          tc_commit_by(&s.empty[slot], leader);
        }
        if (!ok) break;
        tc_commit_by(&s.w_empty[buf], leader);
      }
      if (ok) tc_commit_by(&s.v_done, leader);
    } else {
      // epilogue warps: TMEM lanes 32 quad .. (keys, then dims), rows 16 cg ..
      const uint32_t quad = warp & 3, cg = warp >> 2;
      if (tid < kPtRows) {
        s.top[tid] = INT32_MIN;
        s.query[tid] = tid < rows ? (int32_t)((f0 + tid) / group) : -1;
        s.wsum[tid] = 0;
      }
      epi_sync();
      // 1. scores
      int32_t best[16];
#pragma unroll
      for (uint32_t c = 0; c < 16; ++c) best[c] = INT32_MIN;
      for (uint32_t kt = 0; kt < ktiles && ok; ++kt, ++n_s) {
        if (!tc_wait(&s.s_done, n_s & 1, &s.dead, fault)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t lo[16];
        int32_t hi[16];
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          uint32_t v[5][8];
#pragma unroll
          for (uint32_t d = 0; d < 5; ++d)
            tmem_ld8(tmem + ((32 * quad) << 16) + ((n_s & 1) * 3 + d) * kPtRows + cg * 16 + h * 8, v[d]);
          tmem_ld_wait();
#pragma unroll
          for (uint32_t c = 0; c < 8; ++c) {
            const int32_t x[5] = {(int32_t)v[0][c], (int32_t)v[1][c], (int32_t)v[2][c], (int32_t)v[3][c],
                                  (int32_t)v[4][c]};
            sum_digits<DC * kPtD>(x, &hi[h * 8 + c], &lo[h * 8 + c]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.t_free);
        const uint32_t key = k0 + kt * kPtKeys + 32 * quad + lane;
        // the warp's keys, seen by every row of the tile?
        const uint32_t kw = k0 + kt * kPtKeys + 32 * quad;
        const bool open = rows == kPtRows && kw + 31 <= begin + q0 && kw >= begin + window_start(q1, a.window);
        int32_t* out = scores + (uint64_t)kt * kPtBlock + cg * 16 * kPtKeys + 32 * quad + lane;
#pragma unroll
        for (uint32_t c = 0; c < 16; ++c) {
          int32_t x = score_of(hi[c], lo[c], a.scale_q32);
          if (!open) {
            const int32_t q = s.query[cg * 16 + c];
            if (q < 0 || key > begin + (uint32_t)q || key < begin + window_start((uint32_t)q, a.window)) x = INT32_MIN;
          }
          best[c] = max(best[c], x);
          __stcg(out + c * kPtKeys, x);
        }
      }
#pragma unroll
      for (uint32_t c = 0; c < 16; ++c) {
        const int32_t x = __reduce_max_sync(0xffffffffu, best[c]);
        if (lane == 0) atomicMax(&s.top[cg * 16 + c], x);
      }
      // After a give-up the scratch holds no scores, and the queries' copies may still
      // be landing under the lists: no row is worked on then.
      ok = epi_all(ok);
      // 2. terms in place, a row a warp (hidden keys: see prompt_mma.cu)
      const uint32_t padded = ktiles * kPtKeys;
      uint32_t* list = (uint32_t*)ops + warp * kPtList;  // (the query planes are done with)
      // eight scores a lane and turn (two key tiles) of a row
      const int4 hidden = make_int4(INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN);
      auto load = [&](int4 (&z)[2], const int32_t* row, uint32_t kt) {
        const int32_t* at = row + (uint64_t)kt * kPtBlock + 4 * lane;
        z[0] = __ldcg((const int4*)at);
        z[1] = kt + 1 < ktiles ? __ldcg((const int4*)(at + kPtBlock)) : hidden;
      };
      int4 x[2];
      load(x, scores + warp * kPtKeys, 0);
      for (uint32_t i = warp; i < kPtRows; i += kPtEpiWarps) {
        const int32_t top = s.top[i], q = ok ? s.query[i] : -1;
        const bool ask = top < INT32_MIN + (1 << 20);
        int32_t* row = scores + i * kPtKeys;  // key t at (t / 128) blocks + t % 128
        uint64_t sum = 0;
        uint32_t first = UINT32_MAX;
        if (q >= 0 && !ask) {
          // the next eight (or the next row's first) are loaded ahead; scores
          // nearer to the maximum than the table goes are put on a list (place
          // and distance in one word) and done 32 at a time, exactly
          int4 y[2] = {hidden, hidden};
          uint32_t listed = 0;
          auto drain = [&] {
            __syncwarp();
            for (uint32_t n = lane; n < listed; n += 32) {
              const uint32_t at = list[n] >> kPtNearBits, d = list[n] & ((1u << kPtNearBits) - 1);
              const uint32_t z = d ? exp_term_near(d) : kTermTop;
              if (!d) first = min(first, at);
              sum += kept_term(z);
              __stcg((uint32_t*)row + (at / kPtKeys) * kPtBlock + at % kPtKeys, z);
            }
            listed = 0;
            __syncwarp();
          };
          for (uint32_t kt = 0; kt < ktiles; kt += 2) {
            if (kt + 2 < ktiles) load(y, row, kt + 2);
            else if (i + kPtEpiWarps < kPtRows) load(y, row + kPtEpiWarps * kPtKeys, 0);
            uint32_t e[8], d[8];
            terms_by_table(x, top, bits, e, d);
            sum += ((uint64_t)e[0] + e[1] + ((uint64_t)e[2] + e[3])) + ((uint64_t)e[4] + e[5] + ((uint64_t)e[6] + e[7]));
            uint32_t* at = (uint32_t*)row + (uint64_t)kt * kPtBlock + 4 * lane;
            __stcg((uint4*)at, make_uint4(e[0], e[1], e[2], e[3]));
            if (kt + 1 < ktiles) __stcg((uint4*)(at + kPtBlock), make_uint4(e[4], e[5], e[6], e[7]));
            const uint32_t least = min(min(min(d[0], d[1]), min(d[2], d[3])), min(min(d[4], d[5]), min(d[6], d[7])));
            if (__any_sync(0xffffffffu, least < kExpExactBelow)) {
              uint32_t near = 0;
#pragma unroll
              for (uint32_t u = 0; u < 8; ++u) near |= (d[u] < kExpExactBelow ? 1u : 0u) << u;
              for (uint32_t who; (who = __ballot_sync(0xffffffffu, near != 0)) != 0; near &= near - 1) {
                if (near) {
                  const uint32_t u = __ffs(near) - 1;
                  uint32_t dist = d[0];
#pragma unroll
                  for (uint32_t o = 1; o < 8; ++o) dist = u == o ? d[o] : dist;
                  list[listed + __popc(who & ((1u << lane) - 1))] =
                      ((kt + u / 4) * kPtKeys + 4 * lane + u % 4) << kPtNearBits | dist;
                }
                listed += __popc(who);
              }
              if (listed + 256 > kPtList) drain();
            }
            x[0] = y[0], x[1] = y[1];
          }
          drain();
        } else {
          if (i + kPtEpiWarps < kPtRows) load(x, row + kPtEpiWarps * kPtKeys, 0);
        }
        if (q >= 0 && ask) {
          // every score within 16.0 of the lowest: hidden keys by their place
          const uint32_t k1 = begin + (uint32_t)q, ks = begin + window_start((uint32_t)q, a.window);
          for (uint32_t t = lane; t < padded; t += 32) {
            int32_t* at = row + (t / kPtKeys) * kPtBlock + t % kPtKeys;
            const uint32_t z = k0 + t < ks || k0 + t > k1 ? 0 : term_of(__ldcg(at), top);
            if (z == kTermTop) first = min(first, t);
            sum += kept_term(z);
            __stcg((uint32_t*)at, z);
          }
        }
        sum = (uint64_t)warp_sum_i64((int64_t)sum);
        first = __reduce_min_sync(0xffffffffu, first);
        __syncwarp();
        if (lane == 0) {
          s.sum[i] = sum;
          s.first[i] = place_within(first, count);
          if (q >= 0 && first < padded) __stcg(row + (first / kPtKeys) * kPtBlock + first % kPtKeys, 0);  // its weight comes last
        }
      }
      __syncwarp();
      if (lane < kPtRows / kPtEpiWarps) {
        const uint32_t i = warp + lane * kPtEpiWarps;
        s.recip[i] = sum_recip(s.sum[i]);
      }
      epi_sync();
      // 3. weights: eight keys of a row a thread, two rows' worth a tile
      int32_t all[2] = {};
      uint4 next[2][2], after[2][2];
      auto load_terms = [&](uint4 (&next)[2][2], uint32_t kt) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          const int32_t* e = scores + (uint64_t)kt * kPtBlock + ((tid >> 4) + 32 * h) * kPtKeys + 8 * (tid & 15);
          next[h][0] = __ldcg((const uint4*)e);
          next[h][1] = __ldcg((const uint4*)(e + 4));
        }
      };
      load_terms(next, 0);
      if (ktiles > 1) load_terms(after, 1);
      for (uint32_t kt = 0; kt < ktiles && ok; ++kt, ++n_w) {
        const uint32_t buf = n_w & 1, use = n_w >> 1;
        if (use > 0 && !tc_wait(&s.w_empty[buf], (use - 1) & 1, &s.dead, fault)) {
          ok = false;
          break;
        }
        uint8_t* wb = ops + buf * kPtWBuf;
        uint4 now[2][2];
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
          for (uint32_t m = 0; m < 2; ++m) now[h][m] = next[h][m], next[h][m] = after[h][m];
        if (kt + 2 < ktiles) load_terms(after, kt + 2);
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
          const uint32_t i = (tid >> 4) + 32 * h, c = tid & 15;
          const uint4 x0 = now[h][0], x1 = now[h][1];
          const uint32_t term[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
          const uint32_t recip = s.recip[i];
          const uint64_t sum = s.sum[i];
          int32_t w[8];
          weights_of(term, recip, sum, w);
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j) all[h] += w[j];
          const uint32_t t0 = __byte_perm(w[0], w[1], 0x5140), t1 = __byte_perm(w[2], w[3], 0x5140);
          const uint32_t u0 = __byte_perm(w[4], w[5], 0x5140), u1 = __byte_perm(w[6], w[7], 0x5140);
          uint8_t* dst = wb + swizzled(i, 8 * c);
          *(uint2*)dst = make_uint2(__byte_perm(t0, t1, 0x5410), __byte_perm(u0, u1, 0x5410));
          *(uint2*)(dst + kPtQPlane) = make_uint2(__byte_perm(t0, t1, 0x7632), __byte_perm(u0, u1, 0x7632));
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.w_full[buf]);
      }
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        int32_t x = all[h];
#pragma unroll
        for (uint32_t o = 1; o <= 8; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if ((lane & 15) == 0) s.wsum[(tid >> 4) + 32 * h] = x;
      }
      // the first maxima's values, ahead of the last products
      int32_t vf[DC][16];
#pragma unroll
      for (uint32_t h = 0; h < DC; ++h)
#pragma unroll
        for (uint32_t c = 0; c < 16; ++c) {
          const uint32_t x = h * kPtD + 32 * quad + lane;
          vf[h][c] = ok && cg * 16 + c < rows && x < a.head_dim
                         ? a.v[(uint64_t)(k0 + s.first[cg * 16 + c]) * a.v_stride + g * a.head_dim + x]
                         : 0;
        }
      epi_sync();
      if (ok && tc_wait(&s.v_done, n_item & 1, &s.dead, fault)) {
        tc_fence_after();
#pragma unroll
        for (uint32_t h = 0; h < DC; ++h) {
          uint32_t v[4][16];
#pragma unroll
          for (uint32_t d = 0; d < 4; ++d) {
            const uint32_t col = tmem + ((32 * quad) << 16) + (4 * h + d) * kPtRows + cg * 16;
            tmem_ld8(col, v[d]);
            tmem_ld8(col + 8, v[d] + 8);
          }
          tmem_ld_wait();
          const uint32_t x = h * kPtD + 32 * quad + lane;
#pragma unroll
          for (uint32_t c = 0; c < 16; ++c) {
            const uint32_t i = cg * 16 + c;
            if (i < rows && x < a.head_dim) {
              const int32_t y[4] = {(int32_t)v[0][c], (int32_t)v[1][c], (int32_t)v[2][c], (int32_t)v[3][c]};
              int64_t total = diagonal_sum(y);
              mac_wide(total, sub_sat(kOneAct, s.wsum[i]), vf[h][c]);
              a.out[(uint64_t)(begin + s.query[i]) * a.out_stride + (g * group + (f0 + i) % group) * a.head_dim + x] =
                  requantize(total);
            }
          }
        }
      } else {
        ok = false;
      }
      tc_fence_before();
    }
    __syncwarp();
  }
  // every issued copy has landed, and every product is done, before the block exits
  if (warp == kPtEpiWarps && lane == 0) {
    if (n_item) mbar_wait_bounded(&s.q_full, (n_item - 1) & 1, fault, kGaveUpServing);
    for (uint32_t i = 0; i < kPtSlots; ++i)
      if (issued[i]) mbar_wait_bounded(&s.full[i], (issued[i] - 1) & 1, fault, kGaveUpServing);
  }
  if (warp == kPtEpiWarps + 1 && s.dead) tc_drain(&s.drained, leader, fault);
  tc_fence_before();
  __syncthreads();
  if (warp == kPtEpiWarps) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

}  // namespace

bool prompt_tc_usable(const IrisPromptAttention& a) {
  return a.head_dim <= 2 * kPtD && a.longest <= kPtLongest && a.tokens >= kPtKeys &&
         (uint64_t)a.tokens * (a.heads / a.kv_heads) < 0x7FFFFFFFull && (uint64_t)a.kv_heads * 3 < 0x7FFFFFFFull &&
         tensor_map_encoder() != nullptr && device_fault_word() != nullptr;
}

size_t prompt_tc_carve(const IrisPromptAttention& a, uint8_t* base, PromptTcScratch* sc) {
  const uint64_t group = a.heads / a.kv_heads, dp = a.head_dim <= kPtD ? kPtD : 2 * kPtD;
  sc->tpitch = (a.tokens + 127) / 128 * 128;
  sc->pack_blocks = 148 * 4;
  sc->flags = 4 * sc->pack_blocks;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = base + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  sc->qp = take((size_t)a.kv_heads * 3 * a.tokens * group * dp);
  sc->kp = take((size_t)a.kv_heads * 3 * a.tokens * dp);
  sc->vt = take((size_t)a.kv_heads * 3 * dp * sc->tpitch);
  sc->exp_bits = (uint32_t*)take((size_t)kPtTable * 4);
  sc->wide = (uint32_t*)take((size_t)sc->flags * 4);
  return at;
}

namespace {

template <uint32_t DC>
cudaError_t launch(const IrisPromptAttention& a, const PromptTcScratch& sc, uint32_t blocks, cudaStream_t stream) {
  constexpr uint64_t DP = DC * kPtD;
  const uint64_t rows = (uint64_t)a.tokens * (a.heads / a.kv_heads), planes = (uint64_t)a.kv_heads * 3;
  CUtensorMap qmap, kmap, vmap;
  if (!make_map(&qmap, sc.qp, DP, rows, planes, DP, rows * DP, kPtRows, 1) ||
      !make_map(&kmap, sc.kp, DP, a.tokens, planes, DP, (uint64_t)a.tokens * DP, kPtKeys, 1) ||
      !make_map(&vmap, sc.vt, sc.tpitch, DP, planes, sc.tpitch, DP * sc.tpitch, kPtD, 1))
    return cudaErrorInvalidValue;
  static std::atomic<bool> allowed[64];
  cudaError_t e = allow_smem(prompt_tc_kernel<DC>, allowed);
  if (e != cudaSuccess) return e;
  e = launch_k(prompt_pack_kernel<DC>, dim3(sc.pack_blocks, 4), dim3(kPackThreads), 0, stream, a, sc);
  if (e != cudaSuccess) return e;
  return launch_k(prompt_tc_kernel<DC>, dim3(blocks), dim3(kPtThreads), PtLayout<DC>::kSmem, stream, a, sc, qmap, kmap,
                  vmap, device_fault_word());
}

}  // namespace

cudaError_t launch_prompt_tc(const IrisPromptAttention& a, const PromptTcScratch& sc, uint32_t blocks,
                             cudaStream_t stream) {
  return a.head_dim <= kPtD ? launch<1>(a, sc, blocks, stream) : launch<2>(a, sc, blocks, stream);
}

}  // namespace iris
