// Pieces of the serving attention kernels on the tcgen05 tensor cores: bounded
// waits, product issue without a branch, signed digits.
#pragma once
#include "common.cuh"
#include "serve_mma.cuh"
#include "tcgen05.cuh"

namespace iris {

// mbar_wait_bounded that gives up at once after any wait of the block has
// (*dead, in shared memory).
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, uint32_t* dead, unsigned int* fault) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (;;) {
    if (mbar_try_wait_suspend(bar, parity)) return true;
    if (*(volatile uint32_t*)dead) return false;
    if (global_ns() - t0 > 1000000000ull) {
      *(volatile uint32_t*)dead = 1;
      atomicOr(fault, kGaveUpServing);
      return false;
    }
  }
}

// tc_mma and tc_commit issued by the lane with `leader`, without a branch.
__device__ __forceinline__ void tc_mma_by(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, bool acc, bool leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"((uint32_t)acc), "r"((uint32_t)leader)
      : "memory");
}
__device__ __forceinline__ void tc_commit_by(uint64_t* bar, bool leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
      "r"((uint32_t)leader)
      : "memory");
}
// After a give-up: waits, with a bound, until the products that this warp issued are
// done (bar: initialised for one arrival, unused before), so that none runs on in
// shared memory and accumulators that the block gives back.
__device__ __forceinline__ void tc_drain(uint64_t* bar, bool leader, unsigned int* fault) {
  tc_commit_by(bar, leader);
  __syncwarp();
  mbar_wait_bounded(bar, 0, fault, kGaveUpServing);
}
// Shared-memory writes of this thread made visible to the tensor cores' reads.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Four values as signed base-256 digits, x = c0 + 2^8 c1 + 2^16 c2 with every
// digit in [-128, 127]: the bytes of x + 0x808080, each less 128. p[3] is not 0
// where a value is outside [-0x808080, 0x7F7F7F]. With all digits signed, one
// product takes a plane against several others side by side.
__device__ __forceinline__ void split_digits(int32_t x, int32_t y, int32_t z, int32_t w, uint32_t (&p)[4]) {
  split_planes(x + 0x808080, y + 0x808080, z + 0x808080, w + 0x808080, p);
#pragma unroll
  for (uint32_t i = 0; i < 3; ++i) p[i] ^= 0x80808080u;
}

// The 64-bit sum of five diagonals of signed digits over D dims: for up to 128,
// two diagonals together are below 2^31 (2^21 + 2^8 2^22, 3 2^21 + 2^8 2^22).
template <uint32_t D>
__device__ __forceinline__ void sum_digits(const int32_t (&v)[5], int32_t* hi, uint32_t* lo) {
  if (D > 128) {
    carry_diagonals(v, hi, lo);
    return;
  }
  const int64_t s = (int64_t)(v[2] + v[3] * 256) * 65536 + (v[0] + v[1] * 256);
  *hi = (int32_t)(s >> 32) + v[4];
  *lo = (uint32_t)s;
}

// Byte offset of byte x of row y in a tile of 128-byte rows in the 128-byte
// swizzle: 16-byte pieces exchanged by the row's low bits.
__device__ __forceinline__ uint32_t swizzled(uint32_t y, uint32_t x) { return y * 128 + (((x >> 4) ^ (y & 7)) << 4) + (x & 15); }

}  // namespace iris
