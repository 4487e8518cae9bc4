// evict.cuh -- the keys of each cache row that stay under a budget, packed in place.
//
// A row with n cached keys and a budget b keeps its m = min(n, b) highest-ranked keys.  The
// rank is a 32-bit whole number: all ones for a protected key (position below `sink`, or
// among the last `recent` positions up to the row's newest), else the order-preserving
// image of the key's weight sum (NaN last); equal ranks go to the lower slot.
//
// Softmax does not see the order of keys, so nothing is shifted: the i-th slot below m whose
// key goes takes the i-th kept key at or beyond m (both in slot order).  At most min(m, n - m)
// keys move, each once, and every move reads at or beyond m and writes below it, so moves
// never meet.
#pragma once

#include "cache_pages.cuh"

namespace hyp {
namespace evict {

constexpr int kThreads = 1024;
constexpr uint32_t kProtected = 0xffffffffu;

struct Args {
  uint32_t* k;  // [pool_rows, D / 32]
  uint8_t* v;   // [pool_rows, D]
  float* v_scale;  // nullptr or [pool_rows]
  int row_words;   // D / 32
  const int32_t* ctx_in;
  int32_t* ctx_out;
  int n_kv;
  Pages pages;
  const float* w_in;
  float* w_out;
  const int32_t* pos_in;
  int32_t* pos_out;
  long long ld;
  const int32_t* keep_rows;  // nullptr: `keep` for every row
  int keep, sink, recent;
  int32_t* holes;  // [n_kv, hole_ld]
  long long hole_ld;
  uint32_t* err;
};

// Order-preserving image of a weight sum: -0 as +0, NaN below everything.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0;
  const uint32_t b = __float_as_uint(w + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Sum of `x` over the lower-numbered threads of the block; *total gets the whole sum.
__device__ __forceinline__ int block_rank(int x, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  __syncthreads();  // the previous use of s_warp is over
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  int before = 0, all = 0;
  for (int j = 0; j < kThreads / 32; ++j) {
    const int y = s_warp[j];
    if (j < warp) before += y;
    all += y;
  }
  *total = all;
  return before + inc - x;
}

__global__ void __launch_bounds__(kThreads) evict_kernel(Args a) {
  __shared__ int s_hist[256];
  __shared__ int s_warp[kThreads / 32];
  __shared__ int s_pick[2];
  const int r = blockIdx.x, tid = threadIdx.x;
  const int n = a.pages.context(a.ctx_in[r], a.err, tid == 0);
  int m = a.keep_rows ? __ldg(a.keep_rows + r) : a.keep;
  m = min(n, max(m, 0));
  const float* w = a.w_in + r * a.ld;
  const int32_t* pos = a.pos_in + r * a.ld;
  float* w_out = a.w_out + r * a.ld;
  int32_t* pos_out = a.pos_out + r * a.ld;
  __syncthreads();  // ctx_out may be ctx_in
  if (tid == 0) a.ctx_out[r] = m;
  if (m == n) {
    for (int t = tid; t < n; t += kThreads) {
      w_out[t] = w[t];
      pos_out[t] = pos[t];
    }
    return;
  }

  int newest = INT_MIN;
  for (int t = tid; t < n; t += kThreads) newest = max(newest, pos[t]);
  newest = __reduce_max_sync(0xffffffffu, newest);
  if ((tid & 31) == 0) s_warp[tid >> 5] = newest;
  __syncthreads();
  for (int j = 0; j < kThreads / 32; ++j) newest = max(newest, s_warp[j]);
  const long long recent_above = (long long)newest - a.recent;
  auto rank = [&](int t) {
    const int p = pos[t];
    return (p < a.sink || (long long)p > recent_above) ? kProtected : rank_of(w[t]);
  };

  // The m-th largest rank, 8 bits a pass from the top; `left` of the ranks equal to it stay.
  uint32_t prefix = 0;
  int left = m;
  for (int shift = 24; shift >= 0 && m > 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
    for (int t = tid; t < n; t += kThreads) {
      const uint32_t x = rank(t);
      if (shift == 24 || (x >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(x >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int need = left, d = 255;
      while (need > s_hist[d]) need -= s_hist[d--];
      s_pick[0] = d;
      s_pick[1] = need;
    }
    __syncthreads();
    prefix |= (uint32_t)s_pick[0] << shift;
    left = s_pick[1];
  }

  // Kept slots in order: the emptied ones below m are listed, those beyond m move into them.
  int32_t* holes = a.holes + r * a.hole_ld;
  int equal_seen = 0, n_holes = 0, n_moved = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int t = base + tid;
    const uint32_t x = t < n ? rank(t) : 0;
    const bool equal = t < n && m > 0 && x == prefix;
    int total;
    const int e = equal_seen + block_rank(equal, s_warp, &total);
    equal_seen += total;
    const bool kept = t < n && m > 0 && (x > prefix || (equal && e < left));
    const int hr = n_holes + block_rank(t < m && !kept, s_warp, &total);
    n_holes += total;
    if (t < m && !kept) holes[hr] = t;
    __syncthreads();  // the holes below m all come before the keys beyond it read them
    const int sr = n_moved + block_rank(t >= m && kept, s_warp, &total);
    n_moved += total;
    if (t >= n) continue;
    if (t < m) {
      if (kept && w_out != w) w_out[t] = w[t];
      if (kept && pos_out != pos) pos_out[t] = pos[t];
      continue;
    }
    if (kept) {
      const int to = holes[sr];
      w_out[to] = w[t];
      pos_out[to] = pos[t];
      const long long src = a.pages.slot(r, t), dst = a.pages.slot(r, to);
      if (src < 0 || dst < 0) {
        raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
      } else {
        const int W = a.row_words;
        for (int i = 0; i < W; ++i) a.k[dst * W + i] = a.k[src * W + i];
        const uint4* vs = reinterpret_cast<const uint4*>(a.v + src * 32 * W);
        uint4* vd = reinterpret_cast<uint4*>(a.v + dst * 32 * W);
        for (int i = 0; i < 2 * W; ++i) vd[i] = vs[i];
        if (a.v_scale) a.v_scale[dst] = a.v_scale[src];
      }
    }
    w_out[t] = 0.f;
    pos_out[t] = -1;
  }
}

inline long long hole_ld(int block_size, int num_blocks) { return (long long)block_size * num_blocks / 2 + 1; }

inline size_t scratch_bytes(long long n_kv, int block_size, int num_blocks) {
  return (size_t)n_kv * hole_ld(block_size, num_blocks) * sizeof(int32_t);
}

inline cudaError_t launch(const Args& a, cudaStream_t st) {
  evict_kernel<<<(unsigned)a.n_kv, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace evict
}  // namespace hyp
