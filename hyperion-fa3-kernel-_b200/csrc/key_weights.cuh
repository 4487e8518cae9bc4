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

#include <algorithm>
#include <cmath>

#include "cache_pages.cuh"

namespace hyp {
namespace kweights {

constexpr int kThreads = 256;

struct Args {
  const uint32_t* q;  // [n_kv * kv_group * seq_q, W]
  const uint32_t* k;  // [pool_rows, W]
  const int32_t* ctx_lens;
  Pages pages;
  int n_kv, kv_group, seq_q;
  const int32_t* q_first;  // nullptr: row 0
  int n_q;
  float inv_sqrt_d;
  int causal;
  float decay;
  const float* in;
  float* out;
  long long ld;
  int2* stats;  // [n_kv * kv_group * n_q]: best popcount distance base and 1 / l
  uint32_t* err;
  long long wait_cycles;  // bound of every device wait: kWaitCycles, shorter only under a test hook
  int fault_stage;        // test hook: the product that blocks leave out, -1 for none
};

// E[j], j = 0..D.
template <int D>
__device__ __forceinline__ void fill_table(float* e, float inv_sqrt_d, int tid, int n) {
  const float step = 2.f * fabsf(inv_sqrt_d);
  for (int j = tid; j <= D; j += n) e[j] = expf(fmaxf(-step * j, kExpClamp));
}

// Sum and carry of three bits in every place (two LOP3).
__device__ __forceinline__ void full_add(uint32_t a, uint32_t b, uint32_t c, uint32_t& sum, uint32_t& carry) {
  sum = a ^ b ^ c;
  carry = (a & b) | (c & (a ^ b));
}

// A query's or key's words, and those of their sums that every distance needs.
template <int W>
struct Words {
  uint32_t x[W];
  uint32_t s3, s4;  // x0 ^ x1 ^ x2 and that ^ x3 (head_dim 128)
  __device__ __forceinline__ void add_up() {
    s3 = x[0] ^ x[1] ^ x[2];
    s4 = s3 ^ x[3];
  }
};

// popcount(q ^ k); `q` comes inverted for a negative inv_sqrt_d, which makes it D minus
// the popcount.  POPC issues at a quarter of the logic operations' rate or less, so the
// words are first added place by place into words of weight 1, 2 and 4: 3 POPC for 4
// words, 4 for 8.
template <int W>
__device__ __forceinline__ int distance(const Words<W>& q, const Words<W>& k) {
  static_assert(W == 4 || W == 8, "head_dim 128 or 256");
  if constexpr (W == 4) {
    const uint32_t a = q.x[0] ^ k.x[0], b = q.x[1] ^ k.x[1], c = q.x[2] ^ k.x[2];
    const uint32_t carry = (a & b) | (c & (a ^ b));
    return __popc(q.s4 ^ k.s4) + 2 * (__popc(carry) + __popc((q.s3 ^ k.s3) & (q.x[3] ^ k.x[3])));
  } else {
    uint32_t s0, c0, s1, c1, s2, c2, t, f;
    full_add(q.x[0] ^ k.x[0], q.x[1] ^ k.x[1], q.x[2] ^ k.x[2], s0, c0);
    full_add(q.x[3] ^ k.x[3], q.x[4] ^ k.x[4], q.x[5] ^ k.x[5], s1, c1);
    full_add(s0, s1, q.x[6] ^ k.x[6], s2, c2);
    const uint32_t x = q.x[7] ^ k.x[7];
    const uint32_t c3 = s2 & x;
    full_add(c0, c1, c2, t, f);
    return __popc(s2 ^ x) + 2 * __popc(t ^ c3) + 4 * (__popc(f) + __popc(t & c3));
  }
}

template <int W>
__device__ __forceinline__ void load_words(Words<W>& k, const uint32_t* p) {
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + i));
    k.x[i] = v.x, k.x[i + 1] = v.y, k.x[i + 2] = v.z, k.x[i + 3] = v.w;
  }
}

// Query row `i` of KV row r: its row in Q and its key end (0: it has none).
__device__ __forceinline__ int query_of(const Args& a, int r, int i, int ctx, long long* q_row) {
  const int g = a.n_q == 1 ? i : i / a.n_q;
  const long long qi = (long long)(a.q_first ? __ldg(a.q_first + r) : 0) + (i - g * a.n_q);
  if (qi < 0 || qi >= a.seq_q) return 0;
  *q_row = ((long long)r * a.kv_group + g) * a.seq_q + qi;
  return a.causal && ctx > qi + 1 ? (int)qi + 1 : ctx;
}

// A query's words, inverted where the best score has the greatest popcount.
template <int W>
__device__ __forceinline__ void load_query(Words<W>& q, const Args& a, long long q_row) {
  load_words<W>(q, a.q + q_row * W);
  const uint32_t flip = a.inv_sqrt_d < 0.f ? 0xffffffffu : 0u;
#pragma unroll
  for (int i = 0; i < W; ++i) q.x[i] ^= flip;
  q.add_up();
}

// ---------------------------------------------------------------------------
// Few queries per row (decode): two streaming kernels.
//
// score_kernel reads the keys once: every (query, key) distance goes to scratch (a byte,
// two at head_dim 256) and the sum of E over a chunk's keys beside it.  sum_kernel adds a
// row's chunk sums up and turns the distances into weights on the running sums.  Both are
// one pass over their chunk with all of a thread's reads in flight, and the second is
// launched as a programmatic dependent of the first.
//
// Where 2 |inv_sqrt_d| D <= 80 (kFlat; 22.6 for 1 / sqrt(128)) no exponential reaches the
// clamp whatever the row's best score, so E is taken relative to distance 0.  Otherwise a
// chunk's sum is relative to the chunk's best distance, which is stored with it.
//
// 512 rows of 2048 to 8192 keys of 128 dims, 4 queries each: 31 us for both, 42 MB of keys
// and 21 MB of sums read or written (2 TB/s).  By the counters 155 warp instructions per 32
// keys and 4 queries in the scores, 12 of them POPC, and 63 in the sums: 15 us of the 31 if
// every issue slot were used, and 50 to 60 % are.  The rest is short blocks (8 keys a thread
// behind a prologue of page entries, queries and the table), barriers, and one kernel after
// the other.  One kernel with a cluster per row, the sums exchanged over distributed shared
// memory: 40 us, for its cluster barriers.
// ---------------------------------------------------------------------------
constexpr int kBatch = 4;       // queries scored together against a key
constexpr int kMaxBatches = 4;  // of one call on this path: 16 queries

template <int D>
struct Dists {  // distances 0..128 in a byte
  using One = uint8_t;
  using Four = uchar4;
  static constexpr uint32_t kOut = 255;  // a key this query does not see; E[kOut] = 0
};
template <>
struct Dists<256> {  // 0..256
  using One = uint16_t;
  using Four = ushort4;
  static constexpr uint32_t kOut = 511;
};

// E with zeros beyond D.
template <int D>
__device__ __forceinline__ void fill_padded_table(float* e, float inv_sqrt_d, int tid, int n) {
  const float step = 2.f * fabsf(inv_sqrt_d);
  for (int j = tid; j <= (int)Dists<D>::kOut; j += n) e[j] = j <= D ? expf(fmaxf(-step * j, kExpClamp)) : 0.f;
}

struct ChunkArgs {
  int chunks;     // per row, of kThreads * U keys
  int batches;
  int dist_ld;    // keys of a row's distances
  void* dist;     // [n_kv, batches, dist_ld] of Four
  int2* part;     // [n_kv, chunks, batches * kBatch]: best distance (0 when flat), sum
};

// Sums of four values over the warp in 6 shuffles instead of 20: each step sends half of
// the values away and keeps the other half.  Lane i < 4 gets the sum of value i (the order
// of the additions is fixed).
__device__ __forceinline__ float warp_sum4(const float (&x)[4], int lane) {
  const bool o1 = lane & 1, o2 = lane & 2;
  float a = (o1 ? x[1] : x[0]) + __shfl_xor_sync(0xffffffffu, o1 ? x[0] : x[1], 1);
  float b = (o1 ? x[3] : x[2]) + __shfl_xor_sync(0xffffffffu, o1 ? x[2] : x[3], 1);
  float y = (o2 ? b : a) + __shfl_xor_sync(0xffffffffu, o2 ? a : b, 2);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  return y;
}

// A block scores kThreads * U * kSteps keys of one row.  The block's page entries, the
// queries and E are staged in shared memory once, their global reads all in flight
// together, so that a key costs one dependent read and few instructions of its own.
// kOne: the block has its whole row.  The distances stay in registers, the sums in shared
// memory, and the block writes the weights itself: one launch, no scratch.
template <int D, bool kFlat, int U, int kSteps, bool kOne>
__global__ void __launch_bounds__(kThreads) score_kernel(Args a, ChunkArgs c) {
  using DD = Dists<D>;
  using One = typename DD::One;
  using Four = typename DD::Four;
  constexpr int W = D / 32;
  constexpr int kWarps = kThreads / 32;
  constexpr int kKeys = kThreads * U * kSteps;
  constexpr uint32_t kNoPage = 0xffffffffu;
  __shared__ float e[DD::kOut + 1];
  __shared__ Words<W> s_q[kMaxBatches * kBatch];
  __shared__ int s_end[kMaxBatches * kBatch];
  __shared__ uint32_t s_row[kKeys + 1];  // first pool row of each page the block touches
  __shared__ int s_best[kWarps][kBatch];
  __shared__ float s_sum[kWarps][kBatch];
  __shared__ float s_inv[kBatch];
  constexpr bool kKeep = kOne || !kFlat;  // distances are looked at again
  if (!kOne) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / c.chunks, chunk = blockIdx.x - r * c.chunks;
  const int k0 = chunk * kKeys;
  // The table's entries do not wait for the context length: they exist up to the capacity.
  const int page0 = (int)a.pages.div.quotient((uint32_t)k0);
  const int pages = (int)a.pages.div.quotient((uint32_t)(min(k0 + kKeys, a.pages.capacity()) - 1)) - page0 + 1;
  const int n = a.pages.context(__ldg(a.ctx_lens + r), a.err, chunk == 0 && tid == 0);
  if (k0 >= n) return;
  bool hidden = k0 + kKeys > n;  // some query does not see some key of the block
  for (int i = tid; i < pages; i += kThreads) {
    const long long at = (long long)r * a.pages.num_blocks + page0 + i;
    const long long id = a.pages.tables ? (long long)__ldg(a.pages.tables + at) : at;
    const bool ok = id >= 0 && id < (long long)a.pages.pool_blocks;
    s_row[i] = ok ? (uint32_t)(id * a.pages.block_size) : kNoPage;
    if (!ok && (page0 + i) * a.pages.block_size < n) {
      raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
      hidden = true;
    }
  }
  const int rows = a.kv_group * a.n_q;
  if (tid < c.batches * kBatch) {
    // Places of the last batch beyond the last query are scored like query 0 and weigh nothing.
    long long q_row = 0;
    s_end[tid] = query_of(a, r, tid < rows ? tid : 0, n, &q_row);
    load_query<W>(s_q[tid], a, q_row);
    hidden = hidden || s_end[tid] < k0 + kKeys;
  }
  if (kFlat) fill_padded_table<D>(e, a.inv_sqrt_d, tid, kThreads);
  else fill_table<D>(e, a.inv_sqrt_d, tid, kThreads);
  const bool masked = __syncthreads_or(hidden);
  const int last = n - 1;

  auto fetch = [&](uint4 (&raw)[U][W / 4], uint32_t& off, int step) {
    off = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = min(k0 + (step * U + u) * kThreads + tid, last);
      const int page = (int)a.pages.div.quotient((uint32_t)t);
      const uint32_t first = s_row[page - page0];
      uint32_t row = first + (uint32_t)(t - page * a.pages.block_size);
      if (masked && first == kNoPage) {
        row = 0;
        off |= 1u << u;
      }
      const uint4* from = reinterpret_cast<const uint4*>(a.k) + (size_t)row * (W / 4);
#pragma unroll
      for (int w = 0; w < W / 4; ++w) raw[u][w] = __ldg(from + w);
    }
  };

  float acc[kOne ? U * kSteps : 1] = {};
  for (int b = 0; b < c.batches; ++b) {
    Words<W> q[kBatch];
    int best[kBatch];
    float l[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      q[i] = s_q[b * kBatch + i];
      l[i] = 0.f;
      best[i] = (int)DD::kOut;
    }
    Four* row = static_cast<Four*>(c.dist) + ((size_t)r * c.batches + b) * c.dist_ld + k0 + tid;
    Four p[kKeep ? U * kSteps : 1];
    uint4 raw[2][U][W / 4];
    uint32_t off[2];
    fetch(raw[0], off[0], 0);
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      if (step + 1 < kSteps) fetch(raw[(step + 1) & 1], off[(step + 1) & 1], step + 1);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint4(&x)[W / 4] = raw[step & 1][u];
        Words<W> k;
#pragma unroll
        for (int w = 0; w < W / 4; ++w) k.x[4 * w] = x[w].x, k.x[4 * w + 1] = x[w].y, k.x[4 * w + 2] = x[w].z, k.x[4 * w + 3] = x[w].w;
        k.add_up();
        uint32_t d[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) d[i] = (uint32_t)distance<W>(q[i], k);
        if (masked) {
          const int t = k0 + (step * U + u) * kThreads + tid;
#pragma unroll
          for (int i = 0; i < kBatch; ++i)
            if ((off[step & 1] >> u & 1) || t >= s_end[b * kBatch + i]) d[i] = DD::kOut;
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (kFlat) l[i] += e[d[i]];
          else best[i] = min(best[i], (int)d[i]);
        }
        Four f;
        f.x = (One)d[0], f.y = (One)d[1], f.z = (One)d[2], f.w = (One)d[3];
        if (!kOne) row[(step * U + u) * kThreads] = f;
        if (kKeep) p[kKeep ? step * U + u : 0] = f;
      }
    }
    if (!kFlat) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        best[i] = __reduce_min_sync(0xffffffffu, best[i]);
        if (lane == 0) s_best[warp][i] = best[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        for (int w = 0; w < kWarps; ++w) best[i] = min(best[i], s_best[w][i]);
#pragma unroll
      for (int u = 0; u < U * kSteps; ++u) {
        const Four f = p[kKeep ? u : 0];
        const uint32_t d[kBatch] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          if (d[i] != (One)DD::kOut) l[i] += e[(int)d[i] - best[i]];
      }
    }
    const float sum = warp_sum4(l, lane);
    if (lane < kBatch) s_sum[warp][lane] = sum;
    __syncthreads();
    if (tid < kBatch) {
      float x = 0.f;
      for (int w = 0; w < kWarps; ++w) x += s_sum[w][tid];
      int m = kFlat ? 0 : (int)DD::kOut;
      if (!kFlat)
        for (int w = 0; w < kWarps; ++w) m = min(m, s_best[w][tid]);
      if (kOne) {
        s_inv[tid] = x > 0.f && b * kBatch + tid < rows ? 1.f / x : 0.f;
      } else {
        c.part[((size_t)r * c.chunks + chunk) * c.batches * kBatch + b * kBatch + tid] = make_int2(m, __float_as_int(x));
      }
    }
    if (kOne) {
      __syncthreads();
      float inv[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) inv[i] = s_inv[i];
#pragma unroll
      for (int u = 0; u < (kOne ? U * kSteps : 0); ++u) {
        const Four f = p[kKeep ? u : 0];
        const uint32_t d[kBatch] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (kFlat) acc[u] = fmaf(e[d[i]], inv[i], acc[u]);
          else if (d[i] != (One)DD::kOut) acc[u] = fmaf(e[(int)d[i] - best[i]], inv[i], acc[u]);
        }
      }
    }
    if (b + 1 < c.batches) __syncthreads();
  }
  if (kOne) {
    const float* in = a.in + r * a.ld;
    float* out = a.out + r * a.ld;
    float x[kOne ? U * kSteps : 1];
#pragma unroll
    for (int u = 0; u < (kOne ? U * kSteps : 0); ++u) x[u] = in[min(u * kThreads + tid, last)];
#pragma unroll
    for (int u = 0; u < (kOne ? U * kSteps : 0); ++u)
      if (u * kThreads + tid < n) out[u * kThreads + tid] = fmaf(a.decay, x[u], acc[u]);
  }
}

// Each thread takes kGroups runs of 4 neighbouring keys, the runs of a block side by side.
template <int D, bool kFlat, int kGroups>
__global__ void __launch_bounds__(kThreads) sum_kernel(Args a, ChunkArgs c, int chunk_keys, int blocks_per_row, bool vec) {
  using DD = Dists<D>;
  constexpr int kSlots = kMaxBatches * kBatch;
  __shared__ float e[DD::kOut + 1];
  __shared__ int s_best[kSlots];
  __shared__ float s_inv[kSlots];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / blocks_per_row;
  const int base = (blockIdx.x - r * blocks_per_row) * kThreads * 4 * kGroups;
  const int n = a.pages.context(__ldg(a.ctx_lens + r), a.err, false);
  if (base >= n) {
    // Even so: this grid ends after the one it depends on.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const float* in = a.in + r * a.ld;
  float x[kGroups][4];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int t = base + (g * kThreads + tid) * 4;
    if (vec && t + 4 <= n) {
      const float4 v = *reinterpret_cast<const float4*>(in + t);
      x[g][0] = v.x, x[g][1] = v.y, x[g][2] = v.z, x[g][3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[g][i] = t + i < n ? in[t + i] : 0.f;
    }
  }
  if (kFlat) fill_padded_table<D>(e, a.inv_sqrt_d, tid, kThreads);
  else fill_table<D>(e, a.inv_sqrt_d, tid, kThreads);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // The row's sums from its chunks', in a fixed order.
  const int rows = a.kv_group * a.n_q, slots = c.batches * kBatch;
  const int chunks = (n + chunk_keys - 1) / chunk_keys;
  if (!kFlat) __syncthreads();
  for (int i = warp; i < slots; i += kThreads / 32) {
    const int2* part = c.part + (size_t)r * c.chunks * slots + i;
    int best = 0;
    if (!kFlat) {
      best = (int)DD::kOut;
      for (int j = lane; j < chunks; j += 32) best = min(best, __ldcg(part + (size_t)j * slots).x);
      best = __reduce_min_sync(0xffffffffu, best);
    }
    float l = 0.f;
    for (int j = lane; j < chunks; j += 32) {
      const int2 p = __ldcg(part + (size_t)j * slots);
      if (kFlat) l += __int_as_float(p.y);
      else if (p.x != (int)DD::kOut) l += __int_as_float(p.y) * e[p.x - best];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) {
      s_best[i] = best;
      s_inv[i] = l > 0.f && i < rows ? 1.f / l : 0.f;
    }
  }
  constexpr int kWords = sizeof(typename DD::Four) / 4;
  float sum[kGroups][4] = {};
  for (int b = 0; b < c.batches; ++b) {
    const typename DD::Four* row = static_cast<const typename DD::Four*>(c.dist) + ((size_t)r * c.batches + b) * c.dist_ld;
    uint32_t w[kGroups][4][kWords];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int t = base + (g * kThreads + tid) * 4;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        uint4 v = make_uint4(~0u, ~0u, ~0u, ~0u);  // beyond the row: no chunk has written there
        if (t < n) v = __ldcg(reinterpret_cast<const uint4*>(row + t) + i);
        *reinterpret_cast<uint4*>(&w[g][0][0] + 4 * i) = v;
      }
    }
    if (b == 0) __syncthreads();  // e, s_best and s_inv
    if (base + kThreads * 4 * kGroups > n) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kWords; ++j)
          if (base + (g * kThreads + tid) * 4 + i >= n) w[g][i][j] = kWords == 1 ? 0xFFFFFFFFu : DD::kOut * 0x10001u;
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const float inv = s_inv[b * kBatch + q];
      const int best = kFlat ? 0 : s_best[b * kBatch + q];
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t d = kWords == 1 ? __byte_perm(w[g][i][0], 0, 0x4440 + q)
                                         : __byte_perm(w[g][i][q / 2 % kWords], 0, q % 2 ? 0x4432 : 0x4410);
          if (kFlat) sum[g][i] = fmaf(e[d], inv, sum[g][i]);
          else if (d != DD::kOut) sum[g][i] = fmaf(e[(int)d - best], inv, sum[g][i]);
        }
    }
  }
  float* out = a.out + r * a.ld;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int t = base + (g * kThreads + tid) * 4;
    if (vec && t + 4 <= n) {
      *reinterpret_cast<float4*>(out + t) =
          make_float4(fmaf(a.decay, x[g][0], sum[g][0]), fmaf(a.decay, x[g][1], sum[g][1]),
                      fmaf(a.decay, x[g][2], sum[g][2]), fmaf(a.decay, x[g][3], sum[g][3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i < n) out[t + i] = fmaf(a.decay, x[g][i], sum[g][i]);
    }
  }
}

// ---------------------------------------------------------------------------
// Many queries at a scale beyond kFlat: two kernels on the CUDA cores, with each query's
// best and 1 / l between them.  (At the usual scales: key_weights_window.cuh.)  Every pair's
// popcount is taken three times, from words in L1: 32 rows of 256 queries and up to 16384
// keys 940 us, where the tensor-core form takes 90.
// ---------------------------------------------------------------------------
// One block per query row: the least distance and the sum of E over its keys.
template <int D>
__global__ void __launch_bounds__(kThreads) window_stats_kernel(Args a) {
  constexpr int W = D / 32;
  __shared__ float e[D + 1];
  __shared__ int s_min[kThreads / 32];
  __shared__ float s_sum[kThreads / 32];
  fill_table<D>(e, a.inv_sqrt_d, threadIdx.x, kThreads);
  const int rows = a.kv_group * a.n_q;
  const long long id = blockIdx.x;
  const int r = (int)(id / rows);
  const int i = (int)(id - (long long)r * rows);
  const int ctx = a.pages.context(__ldg(a.ctx_lens + r), a.err, i == 0 && threadIdx.x == 0);
  long long q_row = 0;
  const int end = query_of(a, r, i, ctx, &q_row);
  __syncthreads();
  Words<W> q;
  if (end > 0) load_query<W>(q, a, q_row);
  int best = D + 1;
  for (int t = threadIdx.x; t < end; t += kThreads) {
    const long long slot = a.pages.slot(r, t);
    if (slot < 0) {
      raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
      continue;
    }
    Words<W> k;
    load_words<W>(k, a.k + slot * W);
    k.add_up();
    best = min(best, distance<W>(q, k));
  }
  best = __reduce_min_sync(0xffffffffu, best);
  if ((threadIdx.x & 31) == 0) s_min[threadIdx.x >> 5] = best;
  __syncthreads();
  for (int j = 0; j < kThreads / 32; ++j) best = min(best, s_min[j]);
  float l = 0.f;
  for (int t = threadIdx.x; t < end; t += kThreads) {
    const long long slot = a.pages.slot(r, t);
    if (slot < 0) continue;
    Words<W> k;
    load_words<W>(k, a.k + slot * W);
    k.add_up();
    l += e[distance<W>(q, k) - best];
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
__global__ void __launch_bounds__(kThreads) window_sum_kernel(Args a, int blocks_per_row) {
  constexpr int W = D / 32;
  __shared__ float e[D + 1];
  fill_table<D>(e, a.inv_sqrt_d, threadIdx.x, kThreads);
  __syncthreads();
  const int r = blockIdx.x / blocks_per_row;
  const long long t = (long long)(blockIdx.x - r * blocks_per_row) * kThreads + threadIdx.x;
  const int ctx = a.pages.context(__ldg(a.ctx_lens + r), a.err, false);
  if (t >= ctx) return;
  float sum = 0.f;
  const long long slot = a.pages.slot(r, (int)t);
  if (slot >= 0) {
    Words<W> k;
    load_words<W>(k, a.k + slot * W);
    k.add_up();
    const int rows = a.kv_group * a.n_q;
    for (int i = 0; i < rows; ++i) {
      long long q_row = 0;
      if (t >= query_of(a, r, i, ctx, &q_row)) continue;
      Words<W> q;
      load_query<W>(q, a, q_row);
      const int2 st = __ldg(a.stats + (long long)r * rows + i);
      sum += e[distance<W>(q, k) - st.x] * __int_as_float(st.y);
    }
  }
  a.out[r * a.ld + t] = fmaf(a.decay, a.in[r * a.ld + t], sum);
}

}  // namespace kweights
}  // namespace hyp
