// Exact integer attention on the int8 matrix instructions, for operands read
// as they lie in memory (int32 rows): the pieces the serving kernels share.
//
// A Q16.16 value of 24 bits (|x| < 128.0) is three byte planes, x = b0 + 2^8 b1
// + 2^16 b2 with b0, b1 unsigned and b2 signed; a wider one has a fourth, b2
// then unsigned and b3 signed. A dot product is the sum over plane pairs (i, j)
// of 2^(8 (i + j)) sum_d a_i[d] b_j[d]; the pairs of equal i + j share one int32
// accumulator (a "diagonal"): nine products into five diagonals for 24-bit
// operands, sixteen into seven otherwise. Diagonals stay exact: at most four
// products of 2^16 a term, over at most 256 head dimensions or kPvKeys
// positions.
//
// mma.sync m16n8k32 takes a lane's operand bytes four at a time along k, which
// is one 16-byte load of four consecutive int32 values, its 4 x 4 bytes
// transposed into plane words by seven byte permutes: so keys go from global
// memory to the matrix unit through registers only, whatever page they lie in.
#pragma once
#include "common.cuh"
#include "layers.cuh"
#include "serve_attn.cuh"

namespace iris {

// d (16 x 8) += a (16 x 32) b (32 x 8); AS, BS: signed bytes.
template <bool AS, bool BS>
__device__ __forceinline__ void mma_i8(int32_t (&d)[4], const uint32_t (&a)[4], const uint2& b) {
#define IRIS_MMA(at, bt)                                                                                 \
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32." at "." bt                                        \
               ".s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                    \
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])                                          \
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y))
  if constexpr (AS && BS) IRIS_MMA("s8", "s8");
  else if constexpr (AS) IRIS_MMA("s8", "u8");
  else if constexpr (BS) IRIS_MMA("u8", "s8");
  else IRIS_MMA("u8", "u8");
#undef IRIS_MMA
}

// The byte planes of four values, byte u of plane p from value u.
__device__ __forceinline__ void split_planes(int32_t x, int32_t y, int32_t z, int32_t w, uint32_t (&p)[4]) {
  const uint32_t t0 = __byte_perm(x, y, 0x5140), t1 = __byte_perm(x, y, 0x7362);
  const uint32_t u0 = __byte_perm(z, w, 0x5140), u1 = __byte_perm(z, w, 0x7362);
  p[0] = __byte_perm(t0, u0, 0x5410);
  p[1] = __byte_perm(t0, u0, 0x7632);
  p[2] = __byte_perm(t1, u1, 0x5410);
  p[3] = __byte_perm(t1, u1, 0x7632);
}
// Non-zero where plane 3 is not the sign extension of plane 2 (a value past 24 bits).
__device__ __forceinline__ uint32_t past_24_bits(const uint32_t (&p)[4]) {
  uint32_t sign;
  asm("prmt.b32 %0, %1, 0, 0xBA98;" : "=r"(sign) : "r"(p[2]));  // each byte's sign bit, eight times
  return p[3] ^ sign;
}

// ---- scores ---------------------------------------------------------------------
//
// Operand b: the query rows of a tile as fragments in shared memory, word pair
// [row / 8][step][plane][lane] (a step is 32 dimensions).
struct QueryTile {
  const uint2* frag;
  uint32_t steps;
  __device__ __forceinline__ uint2 get(uint32_t nt, uint32_t step, uint32_t plane, uint32_t lane) const {
    return frag[((nt * steps + step) * 4 + plane) * 32 + lane];
  }
};

// Writes rows [8 nt, 8 nt + 8) x step of a tile's fragments: this lane's row is
// 8 nt + lane / 4 (src: that row, or NULL for zeros). Returns past_24_bits.
__device__ __forceinline__ uint32_t put_query_fragment(uint2* frag, uint32_t steps, uint32_t nt, uint32_t step,
                                                       uint32_t lane, const int32_t* src) {
  int4 x = make_int4(0, 0, 0, 0), y = x;
  if (src) {
    x = *(const int4*)(src + step * 32 + 4 * (lane & 3));
    y = *(const int4*)(src + step * 32 + 16 + 4 * (lane & 3));
  }
  uint32_t p[4], q[4];
  split_planes(x.x, x.y, x.z, x.w, p);
  split_planes(y.x, y.y, y.z, y.w, q);
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) frag[((nt * steps + step) * 4 + i) * 32 + lane] = make_uint2(p[i], q[i]);
  return past_24_bits(p) | past_24_bits(q);
}

// Diagonals of 16 keys x 8 NT rows. k0, k1: the lane's two keys' rows (keys
// lane / 4 and lane / 4 + 8 of the tile; NULL: zeros), P planes. Returns
// whether a key value was past 24 bits (with P = 3 the diagonals are wrong then).
template <uint32_t P, uint32_t NT>
__device__ __forceinline__ uint32_t key_products(const int32_t* k0, const int32_t* k1, const QueryTile& q, uint32_t nt0,
                                                 uint32_t lane, int32_t (&acc)[NT][2 * P - 1][4]) {
#pragma unroll
  for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
    for (uint32_t d = 0; d < 2 * P - 1; ++d)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) acc[n][d][e] = 0;
  const uint32_t c4 = 4 * (lane & 3);
  const int4 zero = make_int4(0, 0, 0, 0);
  uint32_t wide = 0;
  int4 x[4];
  auto load = [&](uint32_t step) {
    x[0] = k0 ? *(const int4*)(k0 + step * 32 + c4) : zero;
    x[1] = k1 ? *(const int4*)(k1 + step * 32 + c4) : zero;
    x[2] = k0 ? *(const int4*)(k0 + step * 32 + 16 + c4) : zero;
    x[3] = k1 ? *(const int4*)(k1 + step * 32 + 16 + c4) : zero;
  };
  load(0);
#pragma unroll 1
  for (uint32_t step = 0; step < q.steps; ++step) {
    uint32_t a[4][4];  // [plane][fragment word]
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      uint32_t p[4];
      split_planes(x[i].x, x[i].y, x[i].z, x[i].w, p);
      if (P == 3) wide |= past_24_bits(p);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) a[j][i] = p[j];
    }
    if (step + 1 < q.steps) load(step + 1);
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
#pragma unroll
      for (uint32_t j = 0; j < P; ++j) {
        const uint2 b = q.get(nt0 + n, step, j, lane);
#pragma unroll
        for (uint32_t i = 0; i < P; ++i) {
          if (i + 1 < P && j + 1 < P) mma_i8<false, false>(acc[n][i + j], a[i], b);
          else if (i + 1 < P) mma_i8<false, true>(acc[n][i + j], a[i], b);
          else if (j + 1 < P) mma_i8<true, false>(acc[n][i + j], a[i], b);
          else mma_i8<true, true>(acc[n][i + j], a[i], b);
        }
      }
    }
  }
  return wide;
}

// The score of a sum hi 2^32 + lo, by scale or without (0); sums of 24-bit
// operands stay below 2^62.
template <bool kAny = false>
__device__ __forceinline__ int32_t score_of(int32_t hi, uint32_t lo, uint32_t scale) {
  return scale ? score_by<true, kAny>(hi, lo, scale) : score_by<false, kAny>(hi, lo, scale);
}
template <uint32_t N>
__device__ __forceinline__ void scores_of(const int32_t (&hi)[N], const uint32_t (&lo)[N], uint32_t scale, int32_t (&y)[N]) {
  if (scale) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) y[i] = score_by<true, false>(hi[i], lo[i], scale);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) y[i] = score_by<false, false>(hi[i], lo[i], scale);
  }
}
// Five diagonals: carried byte by byte, the low 32 bits from the bytes left behind.
__device__ __forceinline__ void carry_diagonals(const int32_t (&v)[5], int32_t* hi, uint32_t* lo) {
  const int32_t y = v[1] + (v[0] >> 8), z = v[2] + (y >> 8), u = v[3] + (z >> 8);
  *hi = v[4] + (u >> 8);
  *lo = __byte_perm(__byte_perm(v[0], y, 0x0040), __byte_perm(z, u, 0x0040), 0x5410);
}
__device__ __forceinline__ int32_t diagonal_score(const int32_t (&v)[5], uint32_t scale) {
  int32_t hi;
  uint32_t lo;
  carry_diagonals(v, &hi, &lo);
  return score_of(hi, lo, scale);
}
// Seven: the sum wraps at 64 bits, as the definition's does.
__device__ __forceinline__ int32_t diagonal_score(const int32_t (&v)[7], uint32_t scale) {
  uint64_t s = 0;
#pragma unroll
  for (uint32_t d = 0; d < 7; ++d) s += (uint64_t)(int64_t)v[d] << (8 * d);
  return score_of<true>((int32_t)(s >> 32), (uint32_t)s, scale);
}

template <uint32_t NT>
static __device__ __noinline__ void wide_key_scores(const int32_t* k0, const int32_t* k1, const QueryTile& q,
                                                    uint32_t nt0, uint32_t lane, uint32_t scale, int32_t (&s)[NT][4]) {
#pragma unroll 1
  for (uint32_t n = 0; n < NT; ++n) {
    int32_t acc[1][7][4];
    key_products<4, 1>(k0, k1, q, nt0 + n, lane, acc);
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      const int32_t v[7] = {acc[0][0][e], acc[0][1][e], acc[0][2][e], acc[0][3][e],
                            acc[0][4][e], acc[0][5][e], acc[0][6][e]};
      s[n][e] = diagonal_score(v, scale);
    }
  }
}

// Scores of 16 keys against rows [8 nt0, 8 nt0 + 8 NT) of a tile: the lane's four
// elements of each n are row 8 (nt0 + n) + 2 (lane % 4) + (e & 1), key lane / 4 +
// 8 (e >> 1).
template <uint32_t NT>
__device__ __forceinline__ void key_scores(const int32_t* k0, const int32_t* k1, const QueryTile& q, bool q_wide,
                                           uint32_t nt0, uint32_t lane, uint32_t scale, int32_t (&s)[NT][4]) {
  if (!q_wide) {
    int32_t acc[NT][5][4];
    const uint32_t wide = key_products<3, NT>(k0, k1, q, nt0, lane, acc);
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        const int32_t v[5] = {acc[n][0][e], acc[n][1][e], acc[n][2][e], acc[n][3][e], acc[n][4][e]};
        s[n][e] = diagonal_score(v, scale);
      }
    if (!__any_sync(0xffffffffu, wide != 0)) return;
  }
  wide_key_scores<NT>(k0, k1, q, nt0, lane, scale, s);
}

// ---- weights ----------------------------------------------------------------------
//
// Terms are kept in 32 bits: softmax_exp_term is below 2^32 except at distance
// 0, where it is exactly 2^32; that one is kept as 0xFFFFFFFF (distance 1 gives
// 2^32 - 65536, so no other distance does).
constexpr uint32_t kTermTop = 0xFFFFFFFFu;
__device__ __forceinline__ uint64_t kept_term(uint32_t t) { return t == kTermTop ? kOneQ32 : (uint64_t)t; }

__device__ __forceinline__ uint32_t term_of(int32_t score, int32_t top) {
  const uint32_t d = (uint32_t)top - (uint32_t)score;  // top >= score: the distance, below 2^32
  if (d >= (1u << 20)) return 0;
  return d ? exp_term_near(d) : kTermTop;
}

// A warp turns the scores of a row into their terms, in place: key t lies at row +
// (t / 128) * block + t % 128, keys from `count` on are hidden, terms are written
// up to `stored` (both multiples of 4). Eight scores a lane and turn, with the
// next eight loaded ahead (x holds the first on entry; then those of `next`,
// where that is not NULL). Terms whose estimate is in doubt - the few keys near
// the maximum, and hardly any far from it - go on a list (place and distance in
// one word) and are done 32 at a time, exactly. Returns this lane's part of the
// sum and the first place of the maximum.
constexpr uint32_t kTermList = 512;    // words of shared memory a warp
constexpr uint32_t kTermTiles = 32;    // key tiles that a list's places reach over
struct RowTerms {
  uint64_t sum;
  uint32_t first;
};
__device__ __forceinline__ void row_load(int4 (&z)[2], const int32_t* row, uint32_t block, uint32_t kt, uint32_t count,
                                         uint32_t lane) {
  const int32_t* at = row + (uint64_t)kt * block + 4 * lane;
  const uint32_t t = kt * 128 + 4 * lane;
  const int4 hidden = make_int4(INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN);
  z[0] = t < count ? __ldcg((const int4*)at) : hidden;
  z[1] = t + 128 < count ? __ldcg((const int4*)(at + block)) : hidden;
}
__device__ __forceinline__ RowTerms row_terms(int32_t* row, uint32_t block, uint32_t count, uint32_t stored, int32_t top,
                                              uint32_t* list, uint32_t lane, int4 (&x)[2], const int32_t* next) {
  RowTerms out{0, UINT32_MAX};
  uint32_t listed = 0, base = 0;
  auto drain = [&] {
    __syncwarp();
    for (uint32_t n = lane; n < listed; n += 32) {
      const uint32_t at = base * 128 + (list[n] >> 20), d = list[n] & ((1u << 20) - 1);
      const uint32_t z = d ? exp_term_near(d) : kTermTop;
      if (!d) out.first = min(out.first, at);
      out.sum += kept_term(z);
      __stcg((uint32_t*)row + (uint64_t)(at / 128) * block + at % 128, z);
    }
    listed = 0;
    __syncwarp();
  };
  const uint32_t tiles = (max(count, stored) + 127) / 128;
  for (uint32_t kt = 0; kt < tiles; kt += 2) {
    if (kt - base + 2 > kTermTiles) {
      drain();
      base = kt;
    }
    int4 y[2];
    if (kt + 2 < tiles) row_load(y, row, block, kt + 2, count, lane);
    else if (next) row_load(y, next, block, 0, count, lane);
    const int32_t v[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
    uint32_t e[8], d[8], doubts = 0;
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u) {
      d[u] = (uint32_t)top - (uint32_t)v[u];
      bool doubt;
      const uint32_t z = exp_term_estimate(d[u], &doubt);
      const bool some = d[u] < kExpTerms;
      e[u] = some && !doubt ? z : 0;
      doubts |= (some && doubt ? 1u : 0u) << u;
    }
    out.sum += ((uint64_t)e[0] + e[1] + ((uint64_t)e[2] + e[3])) + ((uint64_t)e[4] + e[5] + ((uint64_t)e[6] + e[7]));
    const uint32_t t = kt * 128 + 4 * lane;
    uint32_t* at = (uint32_t*)row + (uint64_t)kt * block + 4 * lane;
    if (t < stored) __stcg((uint4*)at, make_uint4(e[0], e[1], e[2], e[3]));
    if (t + 128 < stored) __stcg((uint4*)(at + block), make_uint4(e[4], e[5], e[6], e[7]));
    for (uint32_t who; (who = __ballot_sync(0xffffffffu, doubts != 0)) != 0; doubts &= doubts - 1) {
      if (doubts) {
        const uint32_t u = __ffs(doubts) - 1;
        uint32_t dist = d[0];
#pragma unroll
        for (uint32_t o = 1; o < 8; ++o) dist = u == o ? d[o] : dist;
        list[listed + __popc(who & ((1u << lane) - 1))] = ((kt - base + u / 4) * 128 + 4 * lane + u % 4) << 20 | dist;
      }
      listed += __popc(who);
    }
    if (listed + 256 > kTermList) drain(), base = kt + 2;
    x[0] = y[0], x[1] = y[1];
  }
  drain();
  return out;
}

// A row's divisor: floor(2^63 / sum) (at most 2^31: the maximum's own term makes
// the sum at least 2^32); 0 where nothing is seen.
__device__ __forceinline__ uint32_t sum_recip(uint64_t sum) { return sum ? (uint32_t)(((uint64_t)1 << 63) / sum) : 0; }

// The weight of a term (attention_softmax_raw_weight, ops.rs:269-271:
// requantize of the quotient rounded to Q32.32). y = floor(term recip / 2^32)
// lies in (v - 2.5, v] for v = 2^15 times the exact weight (each of the two
// floors takes less than 1, the kept top term less than 1/2), and rounding the
// quotient first moves v by at most 1/4: so the weight is (y + 2^14) >> 15
// unless a multiple of 2^15 lies within 1/4 below or 2.75 above y + 2^14;
// there (4 values of 32768) the two sides of that multiple are told apart
// exactly. Eight weights of one row, the doubtful ones found together.
__device__ __forceinline__ void weights_of(const uint32_t (&term)[8], uint32_t recip, uint64_t sum, int32_t (&w)[8]) {
  uint32_t least = 0x7FFF;
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) {
    const uint32_t y = __umulhi(term[j], recip) + (1u << 14);
    least = min(least, (y + 3) & 0x7FFF);
    w[j] = (int32_t)(y >> 15);
  }
  if (least <= 3) {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint32_t y = __umulhi(term[j], recip) + (1u << 14) + 3;
      if ((y & 0x7FFF) <= 3)
        w[j] = (int32_t)(y >> 15) - !softmax_weight_reaches((int64_t)kept_term(term[j]), sum, y >> 15);
    }
  }
}
// ---- value sums ---------------------------------------------------------------------
//
// sum_t w_t v_t with the first maximum's weight left out (it takes the residual
// and is added last): every other weight is at most 32768, two byte planes.
// Operand a: values, the M rows are 16 head dimensions (dimension 2 g of the
// tile in row g, 2 g + 1 in row g + 8), k 32 positions; operand b: weights, word
// pair [step][row / 8][plane][lane] in shared memory.
constexpr uint32_t kPvKeys = 16384;  // positions an int32 diagonal holds (2 * 255 * 255 * kPvKeys < 2^31)

// acc += 32 positions: v points at the lane's eight rows (positions 4 (lane %
// 4) + i and 16 + 4 (lane % 4) + i), already at the lane's two dimensions.
template <uint32_t P, uint32_t NT>
__device__ __forceinline__ uint32_t value_products(const int2 (&x)[8], const uint2* w, uint32_t lane,
                                                   int32_t (&acc)[NT][P + 1][4]) {
  uint32_t a[4][4], p[4], wide = 0;
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h) {
    split_planes(x[4 * h].x, x[4 * h + 1].x, x[4 * h + 2].x, x[4 * h + 3].x, p);
    if (P == 3) wide |= past_24_bits(p);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) a[j][2 * h] = p[j];
    split_planes(x[4 * h].y, x[4 * h + 1].y, x[4 * h + 2].y, x[4 * h + 3].y, p);
    if (P == 3) wide |= past_24_bits(p);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) a[j][2 * h + 1] = p[j];
  }
#pragma unroll
  for (uint32_t n = 0; n < NT; ++n) {
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint2 b = w[(n * 2 + j) * 32 + lane];
#pragma unroll
      for (uint32_t i = 0; i < P; ++i) {
        if (i + 1 < P) mma_i8<false, false>(acc[n][i + j], a[i], b);
        else mma_i8<true, false>(acc[n][i + j], a[i], b);
      }
    }
  }
  return wide;
}

// A value fragment (16 dimensions x 32 positions) made once for all the warps
// that take it: planes [plane][lane] of four words. Returns past_24_bits.
template <uint32_t P>
__device__ __forceinline__ uint32_t put_value_fragment(uint4* frag, const int2 (&x)[8], uint32_t lane) {
  uint32_t p[4], q[4], r[4], t[4];
  split_planes(x[0].x, x[1].x, x[2].x, x[3].x, p);
  split_planes(x[0].y, x[1].y, x[2].y, x[3].y, q);
  split_planes(x[4].x, x[5].x, x[6].x, x[7].x, r);
  split_planes(x[4].y, x[5].y, x[6].y, x[7].y, t);
#pragma unroll
  for (uint32_t i = 0; i < P; ++i) frag[i * 32 + lane] = make_uint4(p[i], q[i], r[i], t[i]);
  return P == 3 ? past_24_bits(p) | past_24_bits(q) | past_24_bits(r) | past_24_bits(t) : 0;
}
// acc += that fragment against the weights of 8 NT rows.
template <uint32_t P, uint32_t NT>
__device__ __forceinline__ void fragment_products(const uint4* frag, const uint2* w, uint32_t lane,
                                                  int32_t (&acc)[NT][P + 1][4]) {
  uint32_t a[P][4];
#pragma unroll
  for (uint32_t i = 0; i < P; ++i) {
    const uint4 v = frag[i * 32 + lane];
    a[i][0] = v.x, a[i][1] = v.y, a[i][2] = v.z, a[i][3] = v.w;
  }
#pragma unroll
  for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint2 b = w[(n * 2 + j) * 32 + lane];
#pragma unroll
      for (uint32_t i = 0; i < P; ++i) {
        if (i + 1 < P) mma_i8<false, false>(acc[n][i + j], a[i], b);
        else mma_i8<true, false>(acc[n][i + j], a[i], b);
      }
    }
}

// The lane's fragment words of eight weights (positions 4 c .. 4 c + 3 and 16 +
// 4 c ..) of one row: both planes.
__device__ __forceinline__ void put_weight_fragment(uint2* w, uint32_t lane, const int32_t (&x)[8]) {
  const uint32_t t0 = __byte_perm(x[0], x[1], 0x5140), t1 = __byte_perm(x[2], x[3], 0x5140);
  const uint32_t u0 = __byte_perm(x[4], x[5], 0x5140), u1 = __byte_perm(x[6], x[7], 0x5140);
  w[lane] = make_uint2(__byte_perm(t0, t1, 0x5410), __byte_perm(u0, u1, 0x5410));
  w[32 + lane] = make_uint2(__byte_perm(t0, t1, 0x7632), __byte_perm(u0, u1, 0x7632));
}

template <uint32_t ND>
__device__ __forceinline__ int64_t diagonal_sum(const int32_t (&v)[ND]) {
  int64_t s = 0;
#pragma unroll
  for (uint32_t d = 0; d < ND; ++d) s += (int64_t)v[d] << (8 * d);
  return s;
}

// One warp's 16 dimensions over the 32-key steps first, first + by, .. < steps,
// values straight from their pages (v: the lane's two dimensions; row_s: the
// keys' pool rows; w: the steps' weights): emit(row, dimension of the 16, sum) for
// 8 NT rows. Returns whether a value was past 24 bits (P = 3: nothing was
// emitted then).
template <uint32_t P, uint32_t NT, class Emit>
__device__ __forceinline__ bool paged_value_sums(const int32_t* v, size_t kvd, const uint32_t* row_s, const uint2* w,
                                                 uint32_t first, uint32_t by, uint32_t steps, uint32_t lane,
                                                 const Emit& emit) {
  int32_t acc[NT][P + 1][4] = {};
  int2 x[8], y[8];
  auto load = [&](int2 (&z)[8], uint32_t st) {
    const uint32_t* row = row_s + st * 32 + 4 * (lane & 3);
    const uint4 lo = *(const uint4*)row, hi = *(const uint4*)(row + 16);
    const uint32_t r[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) z[i] = *(const int2*)(v + (size_t)r[i] * kvd);
  };
  uint32_t wide = 0;
  if (first < steps) load(x, first);
  for (uint32_t st = first; st < steps; st += by) {
    if (st + by < steps) load(y, st + by);
    wide |= value_products<P, NT>(x, w + (size_t)st * NT * 64, lane, acc);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) x[i] = y[i];
  }
  if (P == 3 && __any_sync(0xffffffffu, wide != 0)) return true;
#pragma unroll
  for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      int32_t d[P + 1];
#pragma unroll
      for (uint32_t j = 0; j < P + 1; ++j) d[j] = acc[n][j][e];
      emit(8 * n + 2 * (lane & 3) + (e & 1), 2 * (lane >> 2) + (e >> 1), diagonal_sum(d));
    }
  return false;
}

}  // namespace iris
