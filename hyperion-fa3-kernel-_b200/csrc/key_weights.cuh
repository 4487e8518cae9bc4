// key_weights.cuh -- the attention weight each cached key receives, summed over query rows.
//
// For KV row r with context length n, and every query row q of its kv_group query heads in
// the call's window,
//   w_q[t] = exp(max(s_t - max s, EXP_CLAMP)) / sum_t exp(...),  s_t = (D - 2 popcount(q ^ k_t)) inv_sqrt_d,
//   out[r][t] = decay * in[r][t] + sum_q w_q[t]      for t < n.
// These are the forward's softmax weights, which it never writes.
//
// A score depends on its popcount alone, so exp(s_t - max s) has at most D + 1 values:
// E[j] = exp(max(-2 |inv_sqrt_d| j, EXP_CLAMP)) at j = the distance of the popcount from
// the row's best one (the least popcount, or the greatest for a negative inv_sqrt_d).  One
// table in shared memory serves every query, scores stay whole numbers, and the row's
// maximum is exact.
#pragma once

#include "common.cuh"

namespace hyp {
namespace kweights {

constexpr int kThreads = 256;

struct Args {
  const uint32_t* q;  // [n_kv * kv_group * seq_q, W]
  const uint32_t* k;  // [pool_rows, W]
  const int32_t* ctx_lens;
  const int32_t* block_tables;
  long long pool_blocks;
  int n_kv, kv_group, seq_q;
  const int32_t* q_first;  // nullptr: row 0
  int n_q;
  int block_size, num_blocks;
  float inv_sqrt_d;
  int causal;
  float decay;
  const float* in;
  float* out;
  long long ld;
  int2* stats;  // [n_kv * kv_group * n_q]: best popcount distance base and 1 / l
  uint32_t* err;
};

// Clamped context length of KV row r; `flag` raises the length's errors.
__device__ __forceinline__ int context_of(const Args& a, int r, bool flag) {
  const int ctx = __ldg(a.ctx_lens + r);
  const long long cap = (long long)a.num_blocks * a.block_size;
  if (ctx < 0) {
    if (flag) raise_error(a.err, HYPERION_DEVERR_NEG_CTX);
    return 0;
  }
  if ((long long)ctx > cap) {
    if (flag) raise_error(a.err, HYPERION_DEVERR_CTX_OVERFLOW);
    return (int)cap;
  }
  return ctx;
}

// Pool row of key t of KV row r, or -1 when its page lies outside the pool.
__device__ __forceinline__ long long slot_of(const Args& a, int r, int t) {
  const int page = t / a.block_size;
  const long long id = a.block_tables ? (long long)__ldg(a.block_tables + (long long)r * a.num_blocks + page)
                                      : (long long)r * a.num_blocks + page;
  if (id < 0 || id >= a.pool_blocks) return -1;
  return id * a.block_size + (t - page * a.block_size);
}

// E[j], j = 0..D.
template <int D>
__device__ __forceinline__ void fill_table(float* e, float inv_sqrt_d, int tid, int n) {
  const float step = 2.f * fabsf(inv_sqrt_d);
  for (int j = tid; j <= D; j += n) e[j] = expf(fmaxf(-step * j, kExpClamp));
}

// popcount(q ^ k), or D minus it when the best score has the greatest popcount.
template <int W>
__device__ __forceinline__ int distance(const uint32_t (&q)[W], const uint32_t (&k)[W], uint32_t flip) {
  int p = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) p += __popc(q[i] ^ k[i] ^ flip);
  return p;
}

template <int W>
__device__ __forceinline__ void load_words(uint32_t (&x)[W], const uint32_t* p) {
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + i));
    x[i] = v.x;
    x[i + 1] = v.y;
    x[i + 2] = v.z;
    x[i + 3] = v.w;
  }
}

// Query row `i` of KV row r: its row in Q and its key end (0: it has none).
__device__ __forceinline__ int query_of(const Args& a, int r, int i, int ctx, long long* q_row) {
  const int g = i / a.n_q;
  const long long qi = (long long)(a.q_first ? __ldg(a.q_first + r) : 0) + (i - g * a.n_q);
  if (qi < 0 || qi >= a.seq_q) return 0;
  *q_row = ((long long)r * a.kv_group + g) * a.seq_q + qi;
  return a.causal && ctx > qi + 1 ? (int)qi + 1 : ctx;
}

// One block per query row: the least distance and the sum of E over its keys.
template <int D>
__global__ void __launch_bounds__(kThreads) stats_kernel(Args a) {
  constexpr int W = D / 32;
  __shared__ float e[D + 1];
  __shared__ int s_min[kThreads / 32];
  __shared__ float s_sum[kThreads / 32];
  fill_table<D>(e, a.inv_sqrt_d, threadIdx.x, kThreads);
  const int rows = a.kv_group * a.n_q;
  const long long id = blockIdx.x;
  const int r = (int)(id / rows);
  const int i = (int)(id - (long long)r * rows);
  const int ctx = context_of(a, r, i == 0 && threadIdx.x == 0);
  long long q_row = 0;
  const int end = query_of(a, r, i, ctx, &q_row);
  const uint32_t flip = a.inv_sqrt_d < 0.f ? 0xffffffffu : 0u;
  __syncthreads();
  uint32_t q[W];
  if (end > 0) load_words<W>(q, a.q + q_row * W);
  int best = D + 1;
  for (int t = threadIdx.x; t < end; t += kThreads) {
    const long long slot = slot_of(a, r, t);
    if (slot < 0) {
      raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
      continue;
    }
    uint32_t k[W];
    load_words<W>(k, a.k + slot * W);
    best = min(best, distance<W>(q, k, flip));
  }
  best = __reduce_min_sync(0xffffffffu, best);
  if ((threadIdx.x & 31) == 0) s_min[threadIdx.x >> 5] = best;
  __syncthreads();
  for (int j = 0; j < kThreads / 32; ++j) best = min(best, s_min[j]);
  float l = 0.f;
  for (int t = threadIdx.x; t < end; t += kThreads) {
    const long long slot = slot_of(a, r, t);
    if (slot < 0) continue;
    uint32_t k[W];
    load_words<W>(k, a.k + slot * W);
    l += e[distance<W>(q, k, flip) - best];
  }
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = l;
  __syncthreads();
  if (threadIdx.x == 0) {
    l = 0.f;
    for (int j = 0; j < kThreads / 32; ++j) l += s_sum[j];
    a.stats[id] = make_int2(best, __float_as_int(l > 0.f ? 1.f / l : 0.f));
  }
}

// One thread per key: the sum over its row's queries.
template <int D>
__global__ void __launch_bounds__(kThreads) sum_kernel(Args a, int blocks_per_row) {
  constexpr int W = D / 32;
  __shared__ float e[D + 1];
  fill_table<D>(e, a.inv_sqrt_d, threadIdx.x, kThreads);
  __syncthreads();
  const int r = blockIdx.x / blocks_per_row;
  const long long t = (long long)(blockIdx.x - r * blocks_per_row) * kThreads + threadIdx.x;
  const int ctx = context_of(a, r, false);
  if (t >= ctx) return;
  const uint32_t flip = a.inv_sqrt_d < 0.f ? 0xffffffffu : 0u;
  float sum = 0.f;
  const long long slot = slot_of(a, r, (int)t);
  if (slot >= 0) {
    uint32_t k[W];
    load_words<W>(k, a.k + slot * W);
    const int rows = a.kv_group * a.n_q;
    for (int i = 0; i < rows; ++i) {
      long long q_row = 0;
      if (t >= query_of(a, r, i, ctx, &q_row)) continue;
      uint32_t q[W];
      load_words<W>(q, a.q + q_row * W);
      const int2 st = __ldg(a.stats + (long long)r * rows + i);
      sum += e[distance<W>(q, k, flip) - st.x] * __int_as_float(st.y);
    }
  }
  a.out[r * a.ld + t] = fmaf(a.decay, a.in[r * a.ld + t], sum);
}

inline size_t scratch_bytes(long long n_kv, int kv_group, int n_q) {
  return (size_t)n_kv * kv_group * n_q * sizeof(int2);
}

template <int D>
inline cudaError_t launch_d(const Args& a, cudaStream_t st) {
  const long long rows = (long long)a.n_kv * a.kv_group * a.n_q;
  const long long cap = (long long)a.num_blocks * a.block_size;
  const int per_row = (int)((cap + kThreads - 1) / kThreads);
  stats_kernel<D><<<(unsigned)rows, kThreads, 0, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  sum_kernel<D><<<(unsigned)(a.n_kv * (long long)per_row), kThreads, 0, st>>>(a, per_row);
  return cudaGetLastError();
}

inline cudaError_t launch(const Args& a, int head_dim, cudaStream_t st) {
  return head_dim == 256 ? launch_d<256>(a, st) : launch_d<128>(a, st);
}

}  // namespace kweights
}  // namespace hyp
