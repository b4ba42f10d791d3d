// Attention of many requests at once: packed prompts (causal, each request on
// its own) and drafted trees over the paged cache. Both are the integer
// attention of the decode loop (attention_softmax ops.rs:233-276 over the
// scores of mistral.rs:130-145 or the unscaled ones, and the weighted value
// sums of tensor.rs:530-536), so a drafted or packed row equals the row that
// decoding the same tokens one at a time gives, bit for bit.
#include <algorithm>

#include "../../include/iris_b200.h"
#include "common.cuh"
#include "layers.cuh"
#include "prompt_mma.cuh"
#include "q8.cuh"
#include "serve.cuh"
#include "serve_attn.cuh"
#include "tree_cluster.cuh"
#include "tree_mma.cuh"

namespace iris {

namespace {

// ---- any head width: a block a (row, query head) --------------------------------
//
// Scores by one thread a key, the first 8192 of them kept in shared memory and
// later ones computed again in each of the three passes (first maximum, sum of
// the terms, weights and value sums). For head widths that are no multiple of 32:
// 512 rows of 8 heads of 80 values 381 us, eight nodes over 777 keys 182 us (heads
// of 128 on the matrix instructions: 93 and 28); bound by its 64-bit products and by
// reading every key once a query head.
constexpr uint32_t kRowThreads = 128, kRowScores = 8192;

struct PackedKeys {
  const int32_t *k, *v;
  uint64_t k_stride, v_stride;
  uint32_t first, n;  // the first key's packed row; keys seen
  __device__ int64_t row(uint32_t j) const { return j < n ? (int64_t)first + j : -1; }
};

struct PagedKeys {
  const int32_t *k, *v;
  uint64_t k_stride, v_stride;
  const int32_t *table, *positions;  // this request's
  uint64_t pages;
  unsigned long long mask;
  uint32_t width, page, held, first, n, window, position;
  __device__ int64_t row(uint32_t j) const {
    const uint32_t at = first + j;
    if (j >= n || !tree_sees(at, held, mask, window, position, positions)) return -1;
    return page_row(table, width, page, pages, at);
  }
};

template <class Keys>
__device__ void attend_row(const Keys& keys, const int32_t* q, int32_t* out, uint32_t g, uint32_t d, uint32_t scale) {
  __shared__ int32_t qs[kServeMaxDim], scores[kRowScores], w_s[kRowThreads];
  __shared__ int64_t row_s[kRowThreads];
  __shared__ unsigned long long best_s[kRowThreads / 32], sum_s[kRowThreads / 32];
  __shared__ int32_t wsum_s[kRowThreads / 32];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (uint32_t i = tid; i < d; i += kRowThreads) qs[i] = q[i];
  __syncthreads();
  auto compute = [&](int64_t row) {
    const int32_t* k = keys.k + (uint64_t)row * keys.k_stride + g * d;
    int64_t acc = 0;
    for (uint32_t i = 0; i < d; i += 4) {
      const int4 x = *(const int4*)(k + i);
      mac_wide(acc, x.x, qs[i]);
      mac_wide(acc, x.y, qs[i + 1]);
      mac_wide(acc, x.z, qs[i + 2]);
      mac_wide(acc, x.w, qs[i + 3]);
    }
    return serve_score(acc, scale);
  };
  auto score = [&](uint32_t j, int64_t row) { return j < kRowScores ? scores[j] : compute(row); };
  unsigned long long best = 0;
  for (uint32_t j = tid; j < keys.n; j += kRowThreads) {
    const int64_t row = keys.row(j);
    if (row < 0) continue;
    const int32_t s = compute(row);
    if (j < kRowScores) scores[j] = s;
    const unsigned long long key = best_key(s, j);
    best = key > best ? key : best;
  }
#pragma unroll
  for (uint32_t o = 16; o >= 1; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, best, o);
    best = x > best ? x : best;
  }
  if (lane == 0) best_s[warp] = best;
  __syncthreads();
  for (uint32_t i = 0; i < kRowThreads / 32; ++i) best = best_s[i] > best ? best_s[i] : best;
  if (!best) {  // nothing is seen
    for (uint32_t i = tid; i < d; i += kRowThreads) out[i] = 0;
    return;
  }
  const int32_t top = best_key_value(best);
  const uint32_t at = best_key_token(best);
  uint64_t sum = 0;
  for (uint32_t j = tid; j < keys.n; j += kRowThreads) {
    const int64_t row = keys.row(j);
    if (row >= 0) sum += (uint64_t)softmax_exp_term_act(score(j, row), top);
  }
  sum = (uint64_t)warp_sum_i64((int64_t)sum);
  if (lane == 0) sum_s[warp] = sum;
  __syncthreads();
  sum = 0;
  for (uint32_t i = 0; i < kRowThreads / 32; ++i) sum += sum_s[i];
  const uint64_t inv = UINT64_MAX / sum;
  int64_t acc[kServeMaxDim / kRowThreads] = {};
  int32_t wsum = 0;
  auto add = [&](uint32_t tiles) {
    for (uint32_t t = 0; t < tiles; ++t) {
      if (row_s[t] < 0) continue;
      const int32_t* v = keys.v + (uint64_t)row_s[t] * keys.v_stride + g * d;
#pragma unroll
      for (uint32_t u = 0; u < kServeMaxDim / kRowThreads; ++u)
        if (tid + u * kRowThreads < d) mac_wide(acc[u], w_s[t], v[tid + u * kRowThreads]);
    }
  };
  for (uint32_t j0 = 0; j0 < keys.n; j0 += kRowThreads) {
    const uint32_t j = j0 + tid;
    const int64_t row = keys.row(j);
    const int32_t w = row < 0 ? 0 : softmax_weight_inv(softmax_exp_term_act(score(j, row), top), sum, inv);
    wsum += w;
    __syncthreads();
    w_s[tid] = w;
    row_s[tid] = row;
    __syncthreads();
    add(min(kRowThreads, keys.n - j0));
  }
  // the residual 1.0 - sum of weights on the first maximum (ops.rs:274-276)
  wsum = (int32_t)warp_sum_i64(wsum);
  if (lane == 0) wsum_s[warp] = wsum;
  __syncthreads();
  if (tid == 0) {
    int32_t all = 0;
    for (uint32_t i = 0; i < kRowThreads / 32; ++i) all += wsum_s[i];
    w_s[0] = sub_sat(kOneAct, all);
    row_s[0] = keys.row(at);
  }
  __syncthreads();
  add(1);
#pragma unroll
  for (uint32_t u = 0; u < kServeMaxDim / kRowThreads; ++u)
    if (tid + u * kRowThreads < d) out[tid + u * kRowThreads] = requantize(acc[u]);
}

__global__ void __launch_bounds__(kRowThreads) prompt_rows_kernel(IrisPromptAttention a) {
  const uint32_t i = blockIdx.x, h = blockIdx.y;
  const uint32_t r = request_of(a.offsets, a.requests, i);
  const uint32_t begin = clamp_offset(a.offsets[r], a.tokens), end = clamp_offset(a.offsets[r + 1], a.tokens);
  if (i < begin || i >= end) return;  // of no request
  const uint32_t at = i - begin, lo = window_start(at, a.window);
  const PackedKeys keys{a.k, a.v, a.k_stride, a.v_stride, begin + lo, at + 1 - lo};
  attend_row(keys, a.q + (uint64_t)i * a.q_stride + h * a.head_dim, a.out + (uint64_t)i * a.out_stride + h * a.head_dim,
             h / (a.heads / a.kv_heads), a.head_dim, a.scale_q32);
}

__global__ void __launch_bounds__(kRowThreads) tree_rows_kernel(IrisTreeAttention a) {
  const uint32_t i = blockIdx.x, h = blockIdx.y;
  const uint32_t r = request_of(a.offsets, a.requests, i);
  const uint32_t begin = clamp_offset(a.offsets[r], a.rows), end = clamp_offset(a.offsets[r + 1], a.rows);
  if (i < begin || i >= end) return;  // of no request
  const uint32_t held = tree_held(a, r), nodes = min(end - begin, kTreeNodes);
  const uint32_t position = a.positions ? (uint32_t)a.positions[i] : 0;
  PagedKeys keys{a.k_pages, a.v_pages, (uint64_t)a.kv_heads * a.head_dim, (uint64_t)a.kv_heads * a.head_dim,
                 a.table + (uint64_t)r * a.width, a.positions ? a.positions + begin : nullptr, a.pages,
                 (unsigned long long)a.masks[i] & node_bits(nodes), a.width, a.page_size, held, 0, 0, a.window, position};
  keys.first = min(held, window_start(position, a.window));
  keys.n = held + nodes - keys.first;
  attend_row(keys, a.q + (uint64_t)i * a.q_stride + h * a.head_dim, a.out + (uint64_t)i * a.out_stride + h * a.head_dim,
             h / (a.heads / a.kv_heads), a.head_dim, a.scale_q32);
}

bool aligned16(const void* p) { return p && ((uintptr_t)p & 15) == 0; }
bool row_stride_ok(uint64_t stride, uint64_t width) { return stride >= width && stride % 4 == 0; }

bool heads_ok(uint32_t heads, uint32_t kv_heads, uint32_t d) {
  return heads && kv_heads && heads <= 65535 && heads % kv_heads == 0 && d && d % 4 == 0 && d <= kServeMaxDim;
}

int check_prompt(const IrisPromptAttention* a) {
  if (!a || !heads_ok(a->heads, a->kv_heads, a->head_dim) || a->tokens > (uint32_t)INT32_MAX) return IRIS_EINVAL;
  if (!a->tokens) return 0;
  const uint64_t qd = (uint64_t)a->heads * a->head_dim, kd = (uint64_t)a->kv_heads * a->head_dim;
  if (!a->requests || !a->offsets || !a->longest || !aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) ||
      !aligned16(a->out) || !row_stride_ok(a->q_stride, qd) || !row_stride_ok(a->k_stride, kd) ||
      !row_stride_ok(a->v_stride, kd) || !row_stride_ok(a->out_stride, qd))
    return IRIS_EINVAL;
  return 0;
}

// No request is longer than all rows together: a looser bound would choose
// kernels and size the scratch for requests that cannot be.
IrisPromptAttention bounded(IrisPromptAttention a) {
  a.longest = std::min(a.longest, a.tokens);
  return a;
}

int check_tree(const IrisTreeAttention* a) {
  if (!a || !heads_ok(a->heads, a->kv_heads, a->head_dim) || a->rows > (uint32_t)INT32_MAX) return IRIS_EINVAL;
  if (!a->rows) return 0;
  const uint64_t qd = (uint64_t)a->heads * a->head_dim;
  if (!a->requests || !a->offsets || !a->held || !a->masks || !a->nodes || a->nodes > kTreeNodes ||
      !a->page_size || a->page_size > (1u << 20) || a->pages > ((uint64_t)1 << 31) || !a->width || !a->table ||
      (a->window && !a->positions) || !aligned16(a->q) || !aligned16(a->k_pages) || !aligned16(a->v_pages) ||
      !aligned16(a->out) || !row_stride_ok(a->q_stride, qd) || !row_stride_ok(a->out_stride, qd) ||
      (uint64_t)a->width * a->page_size > (uint64_t)INT32_MAX || a->longest > (uint64_t)a->width * a->page_size)
    return IRIS_EINVAL;
  return 0;
}

// Positions have 31 bits: a wider window hides nothing, and the kernels add a
// window to an index in 32 bits.
IrisTreeAttention bounded(IrisTreeAttention a) {
  if (a.window > (uint32_t)INT32_MAX) a.window = 0;
  return a;
}

}  // namespace

}  // namespace iris

using namespace iris;

extern "C" {

uint64_t iris_prompt_attention_workspace(const IrisPromptAttention* a) {
  if (check_prompt(a) || !a->tokens) return 0;
  const IrisPromptAttention b = bounded(*a);
  return prompt_mma_usable(b) ? prompt_mma_workspace(b) : 0;
}

int iris_prompt_attention(const IrisPromptAttention* a, void* workspace, uint64_t workspace_bytes, void* stream) {
  const int bad = check_prompt(a);
  if (bad || !a->tokens) return bad;
  const IrisPromptAttention b = bounded(*a);
  const bool mma = prompt_mma_usable(b);
  const uint64_t need = mma ? prompt_mma_workspace(b) : 0;
  if (need && (!aligned16(workspace) || workspace_bytes < need)) return IRIS_ESCRATCH;
  if (mma) return (int)launch_prompt_mma(b, (uint8_t*)workspace, (cudaStream_t)stream);
  prompt_rows_kernel<<<dim3(b.tokens, b.heads), kRowThreads, 0, (cudaStream_t)stream>>>(b);
  return (int)cudaGetLastError();
}

uint64_t iris_tree_attention_workspace(const IrisTreeAttention* a) {
  if (check_tree(a) || !a->rows) return 0;
  const IrisTreeAttention b = bounded(*a);
  return tree_mma_usable(b) && !tree_cluster_usable(b) ? tree_mma_workspace(b) : 0;
}

int iris_tree_attention(const IrisTreeAttention* a, void* workspace, uint64_t workspace_bytes, void* stream) {
  const int bad = check_tree(a);
  if (bad || !a->rows) return bad;
  const IrisTreeAttention b = bounded(*a);
  const bool mma = tree_mma_usable(b), cluster = mma && tree_cluster_usable(b);
  const uint64_t need = mma && !cluster ? tree_mma_workspace(b) : 0;
  if (need && (!aligned16(workspace) || workspace_bytes < need)) return IRIS_ESCRATCH;
  if (cluster) return (int)launch_tree_cluster(b, (cudaStream_t)stream);
  if (mma) return (int)launch_tree_mma(b, (uint8_t*)workspace, (cudaStream_t)stream);
  tree_rows_kernel<<<dim3(b.rows, b.heads), kRowThreads, 0, (cudaStream_t)stream>>>(b);
  return (int)cudaGetLastError();
}

int iris_stall_check(void* stream) {
  uint32_t fault = 0;
  cudaError_t e = cudaStreamSynchronize((cudaStream_t)stream);
  if (e == cudaSuccess) e = take_device_fault(&fault, kGaveUpServing);
  if (e != cudaSuccess) return (int)e;
  return fault ? IRIS_ESTALL : 0;
}

}  // extern "C"
