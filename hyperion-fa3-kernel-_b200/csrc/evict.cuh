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

#include <cooperative_groups.h>

#include <algorithm>

#include "cache_pages.cuh"

namespace hyp {
namespace evict {

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
  int32_t* lists;  // [n_kv, 2, list_ld]: slots that empty below m, kept slots at or beyond it
  long long list_ld;
  uint32_t* err;
};

// Order-preserving image of a weight sum: -0 as +0, NaN below everything.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0;
  const uint32_t b = __float_as_uint(w + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// ---------------------------------------------------------------------------
// The kernel: a cluster of up to 16 blocks per row, each with its part of the row's ranks
// and positions in shared memory.
//
//   1. Read weights and positions once; the row's newest position and the range of its
//      ranks by way of distributed shared memory.
//   2. The m-th largest rank, by histograms of kBins equal intervals of the range that is
//      left: 10 bits a turn, so 3 turns for sums of one sign, fewer when an interval is
//      kept whole.  The blocks add their histograms up over distributed shared memory.
//   3. Each warp walks its neighbouring slots with ballots: counts of slots that empty and
//      of keys that move, then their places in the row's two lists (in slot order).
//   4. The list is dealt evenly to the blocks; D / 16 lanes copy a key's codes 16 bytes each.
// ---------------------------------------------------------------------------
constexpr int kBins = 1024;
constexpr int kMaxCluster = 16;
constexpr int kMovesInFlight = 4;  // keys a lane group copies at once

struct Shared {
  int hist[2][kBins];
  int newest, n_protected;
  uint32_t lo, hi;
  int counts[2];  // slots that empty, keys that move
  // within the block
  int warp_a[32], warp_b[32];
  uint32_t warp_lo[32], warp_hi[32];
  int pick[3];
};

// Exclusive sum over the block's threads of x; *total its whole.  All threads call.
__device__ __forceinline__ int block_scan(int x, int* s_warp, int warps, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  const int w = lane < warps ? s_warp[lane] : 0;
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? w : 0);
  *total = __reduce_add_sync(0xffffffffu, w);
  __syncthreads();
  return before + inc - x;
}

template <int NT>
__global__ void __launch_bounds__(NT) evict_kernel(Args a, int cluster, int keys) {
  namespace cg = cooperative_groups;
  constexpr int kWarps = NT / 32;
  extern __shared__ __align__(16) uint8_t smem[];
  auto& sm = *reinterpret_cast<Shared*>(smem);
  uint32_t* s_rank = reinterpret_cast<uint32_t*>(smem + sizeof(Shared));  // [keys]
  int32_t* s_pos = reinterpret_cast<int32_t*>(s_rank + keys);             // [keys]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / cluster, part = blockIdx.x - r * cluster;
  const int n = a.pages.context(__ldcg(a.ctx_in + r), a.err, part == 0 && tid == 0);
  const int m = min(n, max(a.keep_rows ? __ldg(a.keep_rows + r) : a.keep, 0));
  const int per = ((n + cluster - 1) / cluster + 31) & ~31;
  const int lo = min(part * per, n), len = min(lo + per, n) - lo;
  const float* w = a.w_in + r * a.ld + lo;
  const int32_t* pos = a.pos_in + r * a.ld + lo;
  float* w_out = a.w_out + r * a.ld + lo;
  int32_t* pos_out = a.pos_out + r * a.ld + lo;
  if (m == n) {  // the same for every block of the cluster; writing m changes neither n nor m
    for (int t = tid; t < len; t += NT) {
      if (w_out != w) w_out[t] = w[t];
      if (pos_out != pos) pos_out[t] = pos[t];
    }
    if (part == 0 && tid == 0) a.ctx_out[r] = m;
    return;
  }
  auto all = cg::this_cluster();
  auto sync_all = [&]() {
    if (cluster > 1) all.sync();
    else __syncthreads();
  };
  auto peer = [&](int p) { return cluster > 1 ? all.map_shared_rank(&sm, p) : &sm; };

  // 1. Ranks, positions, newest position, range of the ranks.
  int newest = INT_MIN;
  uint32_t low = 0xffffffffu, high = 0;
#pragma unroll 4
  for (int t = tid; t < len; t += NT) {
    const uint32_t x = rank_of(w[t]);
    const int32_t p = pos[t];
    s_rank[t] = x;
    s_pos[t] = p;
    newest = max(newest, p);
    low = min(low, x);
    high = max(high, x);
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) sm.warp_a[warp] = newest, sm.warp_lo[warp] = low, sm.warp_hi[warp] = high;
  for (int i = tid; i < 2 * kBins; i += NT) (&sm.hist[0][0])[i] = 0;
  __syncthreads();
  if (warp == 0) {
    newest = __reduce_max_sync(0xffffffffu, lane < kWarps ? sm.warp_a[lane] : INT_MIN);
    low = __reduce_min_sync(0xffffffffu, lane < kWarps ? sm.warp_lo[lane] : 0xffffffffu);
    high = __reduce_max_sync(0xffffffffu, lane < kWarps ? sm.warp_hi[lane] : 0u);
    if (lane == 0) sm.newest = newest, sm.lo = low, sm.hi = high, sm.n_protected = 0;
  }
  sync_all();
  {
    const bool on = lane < cluster;
    const Shared* of = peer(on ? lane : 0);
    newest = __reduce_max_sync(0xffffffffu, of->newest);
    low = __reduce_min_sync(0xffffffffu, of->lo);
    high = __reduce_max_sync(0xffffffffu, of->hi);
  }

  // Protected keys rank above every weight; the first histogram comes with the same pass.
  const long long recent_above = (long long)newest - a.recent;
  int shift = max(0, 32 - __clz(high - low) - 10);
  int mine = 0;
  for (int t = tid; t < len; t += NT) {
    const int32_t p = s_pos[t];
    if (p < a.sink || (long long)p > recent_above) {
      s_rank[t] = kProtected;
      ++mine;
    } else {
      atomicAdd(&sm.hist[0][(s_rank[t] - low) >> shift], 1);
    }
  }
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0 && mine) atomicAdd(&sm.n_protected, mine);

  // 2. Kept: rank > top, or rank == top for the first `left` of the row (all when left < 0).
  uint32_t top = kProtected;
  int left = 0, equal_before = 0, need = m;
  for (int turn = 0;; ++turn) {
    sync_all();
    int* hist = sm.hist[turn & 1];
    if (turn == 0) {
      const int p = __reduce_add_sync(0xffffffffu, lane < cluster ? peer(lane < cluster ? lane : 0)->n_protected : 0);
      const int b = __reduce_add_sync(0xffffffffu, lane < part ? peer(lane < cluster ? lane : 0)->n_protected : 0);
      if (m <= p) {
        left = m;
        equal_before = b;
        break;
      }
      need = m - p;
    } else {
      // Nobody reads the other buffer any more.
      for (int i = tid; i < kBins; i += NT) sm.hist[(turn + 1) & 1][i] = 0;
    }
    // This thread's intervals, from the highest down.
    constexpr int kPer = kBins / NT;
    int count[kPer], before[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int bin = kBins - 1 - (tid * kPer + i);
      count[i] = 0;
      for (int p = 0; p < cluster; ++p) count[i] += peer(p)->hist[turn & 1][bin];
      before[i] = sum;
      sum += count[i];
    }
    int total;
    const int above = block_scan(sum, sm.warp_a, kWarps, &total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c0 = above + before[i];
      if (c0 < need && need <= c0 + count[i]) {
        sm.pick[0] = kBins - 1 - (tid * kPer + i);
        sm.pick[1] = need - c0;
        sm.pick[2] = count[i];
      }
    }
    __syncthreads();
    const int bin = sm.pick[0];
    need = sm.pick[1];
    low += (uint32_t)bin << shift;
    if (need == sm.pick[2]) {  // the whole interval stays
      top = low;
      left = -1;
      break;
    }
    if (shift == 0) {
      top = low;
      left = need;
      equal_before = __reduce_add_sync(0xffffffffu, lane < part ? peer(lane < cluster ? lane : 0)->hist[turn & 1][bin] : 0);
      break;
    }
    const uint32_t width = 1u << shift;
    shift = max(0, shift - 10);
    int* next = sm.hist[(turn + 1) & 1];
    for (int t = tid; t < len; t += NT) {
      const uint32_t x = s_rank[t] - low;
      if (s_rank[t] != kProtected && s_rank[t] >= low && x < width) atomicAdd(&next[x >> shift], 1);
    }
    (void)hist;
  }

  // 3. Each warp's neighbouring slots.
  const int seg = ((len + kWarps - 1) / kWarps + 31) & ~31;
  const int w0 = min(warp * seg, len), w1 = min(w0 + seg, len);
  const uint32_t lower = (1u << lane) - 1u;
  if (left >= 0) {
    int eq = 0;
    for (int t = w0 + lane; t < w1; t += 32) eq += s_rank[t] == top;
    eq = __reduce_add_sync(0xffffffffu, eq);
    __syncthreads();
    if (lane == 0) sm.warp_a[warp] = eq;
    __syncthreads();
    equal_before += __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_a[lane] : 0);
  }
  int holes = 0, moved = 0;
  for (int t0 = w0; t0 < w1; t0 += 32) {
    const int t = t0 + lane;
    const uint32_t x = t < w1 ? s_rank[t] : 0;
    bool kept;
    if (left < 0) {
      kept = t < w1 && x >= top;
    } else {
      const uint32_t eq = __ballot_sync(0xffffffffu, t < w1 && x == top);
      kept = t < w1 && (x > top || (x == top && equal_before + __popc(eq & lower) < left));
      equal_before += __popc(eq);
    }
    if (t < w1) s_rank[t] = kept;
    const bool under = lo + t < m;
    holes += __popc(__ballot_sync(0xffffffffu, t < w1 && under && !kept));
    moved += __popc(__ballot_sync(0xffffffffu, kept && !under));
  }
  __syncthreads();
  if (lane == 0) sm.warp_a[warp] = holes, sm.warp_b[warp] = moved;
  __syncthreads();
  int hole_at = __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_a[lane] : 0);
  int move_at = __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_b[lane] : 0);
  if (warp == kWarps - 1 && lane == 0) sm.counts[0] = hole_at + holes, sm.counts[1] = move_at + moved;
  sync_all();
  const Shared* of = peer(lane < cluster ? lane : 0);
  const int c0 = lane < cluster ? of->counts[0] : 0, c1 = lane < cluster ? of->counts[1] : 0;
  hole_at += __reduce_add_sync(0xffffffffu, lane < part ? c0 : 0);
  move_at += __reduce_add_sync(0xffffffffu, lane < part ? c1 : 0);
  const int moves = __reduce_add_sync(0xffffffffu, c1);
  int32_t* empties = a.lists + (size_t)r * 2 * a.list_ld;
  int32_t* movers = empties + a.list_ld;
  for (int t0 = w0; t0 < w1; t0 += 32) {
    const int t = t0 + lane;
    const bool kept = t < w1 && s_rank[t];
    const bool under = lo + t < m;
    const uint32_t h = __ballot_sync(0xffffffffu, t < w1 && under && !kept);
    const uint32_t v = __ballot_sync(0xffffffffu, kept && !under);
    if (t < w1 && under && !kept) empties[hole_at + __popc(h & lower)] = lo + t;
    if (kept && !under) movers[move_at + __popc(v & lower)] = lo + t;
    hole_at += __popc(h);
    move_at += __popc(v);
    if (t < w1) {
      if (under && kept) {
        if (w_out != w) w_out[t] = w[t];
        if (pos_out != pos) pos_out[t] = s_pos[t];
      } else if (!under && !kept) {
        w_out[t] = 0.f;
        pos_out[t] = -1;
      }
    }
  }
  __threadfence();
  sync_all();  // the row's lists; after it no block reads another's shared memory or context length
  if (part == 0 && tid == 0) a.ctx_out[r] = m;

  // 4. The moves [first, last) of this block.
  const int first = (int)((long long)moves * part / cluster), last = (int)((long long)moves * (part + 1) / cluster);
  const int W = a.row_words, G = 2 * W, sub = tid % G, group = tid / G, groups = NT / G;
  const float* w_row = a.w_in + r * a.ld;
  const int32_t* pos_row = a.pos_in + r * a.ld;
  float* w_to = a.w_out + r * a.ld;
  int32_t* pos_to = a.pos_out + r * a.ld;
  for (int i0 = first + group; i0 < last; i0 += groups * kMovesInFlight) {
    int src[kMovesInFlight], dst[kMovesInFlight];
    long long from[kMovesInFlight], to[kMovesInFlight];
#pragma unroll
    for (int u = 0; u < kMovesInFlight; ++u) {
      const int i = min(i0 + u * groups, last - 1);
      src[u] = __ldcg(movers + i);
      dst[u] = __ldcg(empties + i);
    }
#pragma unroll
    for (int u = 0; u < kMovesInFlight; ++u) {
      from[u] = a.pages.slot(r, src[u]);
      to[u] = a.pages.slot(r, dst[u]);
      if (from[u] < 0 || to[u] < 0) {
        if (sub == 0) raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
        from[u] = -1;
      }
    }
    uint4 v[kMovesInFlight], k[kMovesInFlight];
    float wv[kMovesInFlight], sv[kMovesInFlight];
    int32_t pv[kMovesInFlight];
    const bool words = sub < W / 4;
#pragma unroll
    for (int u = 0; u < kMovesInFlight; ++u) {
      const long long at = max(from[u], 0LL);
      v[u] = *(reinterpret_cast<const uint4*>(a.v + at * 32 * W) + sub);
      if (words) k[u] = *(reinterpret_cast<const uint4*>(a.k + at * W) + sub);
      if (sub == 0) {
        wv[u] = w_row[src[u]];
        pv[u] = pos_row[src[u]];
        if (a.v_scale) sv[u] = a.v_scale[at];
      }
    }
#pragma unroll
    for (int u = 0; u < kMovesInFlight; ++u) {
      if (i0 + u * groups >= last) break;
      if (from[u] >= 0) {
        *(reinterpret_cast<uint4*>(a.v + to[u] * 32 * W) + sub) = v[u];
        if (words) *(reinterpret_cast<uint4*>(a.k + to[u] * W) + sub) = k[u];
        if (sub == 0 && a.v_scale) a.v_scale[to[u]] = sv[u];
      }
      if (sub == 0) {
        w_to[dst[u]] = wv[u];
        pos_to[dst[u]] = pv[u];
        w_to[src[u]] = 0.f;
        pos_to[src[u]] = -1;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Rows too long for 16 blocks' shared memory: one block a row, which reads the ranks anew
// for each turn.
// ---------------------------------------------------------------------------
constexpr int kLongThreads = 1024;

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
  for (int j = 0; j < kLongThreads / 32; ++j) {
    const int y = s_warp[j];
    if (j < warp) before += y;
    all += y;
  }
  *total = all;
  return before + inc - x;
}

__global__ void __launch_bounds__(kLongThreads) evict_long_kernel(Args a) {
  __shared__ int s_hist[256];
  __shared__ int s_warp[kLongThreads / 32];
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
    for (int t = tid; t < n; t += kLongThreads) {
      w_out[t] = w[t];
      pos_out[t] = pos[t];
    }
    return;
  }

  int newest = INT_MIN;
  for (int t = tid; t < n; t += kLongThreads) newest = max(newest, pos[t]);
  newest = __reduce_max_sync(0xffffffffu, newest);
  if ((tid & 31) == 0) s_warp[tid >> 5] = newest;
  __syncthreads();
  for (int j = 0; j < kLongThreads / 32; ++j) newest = max(newest, s_warp[j]);
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
    for (int t = tid; t < n; t += kLongThreads) {
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
  int32_t* holes = a.lists + (size_t)r * 2 * a.list_ld;
  int equal_seen = 0, n_holes = 0, n_moved = 0;
  for (int base = 0; base < n; base += kLongThreads) {
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

inline long long list_ld(long long cap) { return cap / 2 + 1; }

inline size_t scratch_bytes(long long n_kv, long long cap) { return (size_t)n_kv * 2 * list_ld(cap) * sizeof(int32_t); }

constexpr size_t kMaxSmem = 227 * 1024;
constexpr int kBlockKeys = 8192;  // of a row per block, while 16 blocks do

inline cudaError_t setup() {
  cudaError_t e = cudaSuccess;
  auto set = [&](const void* kernel) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  };
  set(reinterpret_cast<const void*>(evict_kernel<512>));
  set(reinterpret_cast<const void*>(evict_kernel<1024>));
  return e;
}

inline cudaError_t launch(const Args& a, cudaStream_t st) {
  const long long cap = (long long)a.pages.num_blocks * a.pages.block_size;
  int cluster = 1;
  while (cluster < kMaxCluster && (cap + cluster - 1) / cluster > kBlockKeys) cluster *= 2;
  const long long keys = ((cap + cluster - 1) / cluster + 31) / 32 * 32;
  const size_t smem = sizeof(Shared) + (size_t)keys * 8;
  if (smem > kMaxSmem) {
    evict_long_kernel<<<(unsigned)a.n_kv, kLongThreads, 0, st>>>(a);
    return cudaGetLastError();
  }
  const int threads = keys > 4096 ? 1024 : 512;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)a.n_kv * cluster));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = threads == 1024 ? cudaLaunchKernelEx(&cfg, evict_kernel<1024>, a, cluster, (int)keys)
                                        : cudaLaunchKernelEx(&cfg, evict_kernel<512>, a, cluster, (int)keys);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace evict
}  // namespace hyp
