// Shared pieces of the serving operators: packed rows of several requests and
// the paged K/V cache.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "detnum.cuh"

namespace iris {

// Raises a kernel's dynamic shared memory limit to what a block may have, once
// per device and not on every launch.
template <class K>
inline cudaError_t allow_smem(K* kernel, std::atomic<bool> (&set)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (set[dev].load(std::memory_order_acquire)) return cudaSuccess;
  int most = 0;
  cudaFuncAttributes attr;
  e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, kernel);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)attr.sharedSizeBytes);
  if (e == cudaSuccess) set[dev].store(true, std::memory_order_release);
  return e;
}

constexpr uint32_t kTreeNodes = 64;  // drafted nodes a request: a node's visible nodes are one 64-bit word

// The request r with off[r] <= i < off[r + 1] (off[0] = 0, non-decreasing, i < off[n]).
template <class T>
__device__ __forceinline__ uint32_t request_of(const T* off, uint32_t n, uint32_t i) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if ((uint32_t)off[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// An offset of packed rows, held inside them.
__device__ __forceinline__ uint32_t clamp_offset(int32_t off, uint32_t rows) {
  return min((uint32_t)max(off, 0), rows);
}

// The pool row of a request's position, -1 where its table names no page of the pool.
__device__ __forceinline__ int64_t page_row(const int32_t* table, uint32_t width, uint32_t page, uint64_t pages,
                                            uint32_t at) {
  const uint32_t column = at / page;
  if (column >= width) return -1;
  const int32_t id = table[column];
  return id < 0 || (uint64_t)id >= pages ? -1 : (int64_t)id * page + (at - column * page);
}

}  // namespace iris
