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
  int32_t* counts;  // [n_kv]: moves of each row
  uint32_t* err;
};

// Order-preserving image of a weight sum: -0 as +0, NaN below everything.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0;
  const uint32_t b = __float_as_uint(w + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// ---------------------------------------------------------------------------
// select_kernel: a cluster of up to 16 blocks per row, each with its part of the row's
// ranks in shared memory.
//
//   1. Read weights and positions once; the row's newest position and the range of its
//      ranks by way of distributed shared memory.
//   2. The m-th largest rank, by histograms of kBins equal intervals of the range that is
//      left (10 bits a turn), until an interval is kept whole or holds at most kGather
//      ranks: those are gathered and one warp finds the rank among them bit by bit.  Sums
//      of attention weights take one or two turns.
//   3. A bit per slot says what is kept.  A thread turns a word of 32 slots into its part
//      of the row's two lists (slots that empty below m, keys that move), in slot order.
//
// move_kernel: the moves of all rows, 128 a block, whichever row they belong to.
// ---------------------------------------------------------------------------
constexpr int kBins = 1024;
constexpr int kGather = 256;
constexpr int kMaxCluster = 16;

struct Shared {
  int hist[2][kBins];
  uint32_t cand[kGather];   // this block's ranks of the gathered interval, relative to it
  uint32_t found[kGather];  // the row's
  int n_cand;
  int newest, n_protected;
  uint32_t lo, hi;
  int counts;  // slots that empty | keys that move << 16
  // within the block
  int warp_a[32];
  uint32_t warp_lo[32], warp_hi[32];
  int pick[4];
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

// Bits of word `at` (slots at .. at + 31) that lie below `end`.
__device__ __forceinline__ uint32_t bits_below(int at, int end) {
  const int k = end - at;
  return k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1u;
}

template <int NT, int kBlocks>
__global__ void __launch_bounds__(NT, kBlocks) select_kernel(Args a, int cluster, int keys) {
  namespace cg = cooperative_groups;
  constexpr int kWarps = NT / 32;
  extern __shared__ __align__(16) uint8_t smem[];
  auto& sm = *reinterpret_cast<Shared*>(smem);
  uint32_t* s_rank = reinterpret_cast<uint32_t*>(smem + sizeof(Shared));  // [keys]
  uint32_t* s_kept = s_rank + keys;                                       // [keys / 32]
  uint32_t* s_equal = s_kept + keys / 32;                                 // [keys / 32]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / cluster, part = blockIdx.x - r * cluster;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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
    if (part == 0 && tid == 0) {
      a.ctx_out[r] = m;
      a.counts[r] = 0;
    }
    return;
  }
  auto all = cg::this_cluster();
  auto sync_all = [&]() {
    if (cluster > 1) all.sync();
    else __syncthreads();
  };
  auto peer = [&](int p) { return cluster > 1 ? all.map_shared_rank(&sm, p) : &sm; };
  const int other = lane < cluster ? lane : 0;  // the block whose numbers this lane looks at

  // 1. Ranks, newest position, range of the ranks.
  int newest = INT_MIN;
  uint32_t low = 0xffffffffu, high = 0;
#pragma unroll 4
  for (int t = tid; t < len; t += NT) {
    const uint32_t x = rank_of(w[t]);
    s_rank[t] = x;
    newest = max(newest, pos[t]);
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
    if (lane == 0) sm.newest = newest, sm.lo = low, sm.hi = high, sm.n_protected = 0, sm.n_cand = 0;
  }
  sync_all();
  newest = __reduce_max_sync(0xffffffffu, peer(other)->newest);
  low = __reduce_min_sync(0xffffffffu, peer(other)->lo);
  high = __reduce_max_sync(0xffffffffu, peer(other)->hi);

  // Protected keys rank above every weight; the first histogram comes with the same pass.
  const long long recent_above = (long long)newest - a.recent;
  int shift = max(0, 32 - __clz(high - low) - 10);
  int mine = 0;
#pragma unroll 4
  for (int t = tid; t < len; t += NT) {
    const int32_t p = pos[t];
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
    if (turn == 0) {
      const int x = peer(other)->n_protected;
      const int p = __reduce_add_sync(0xffffffffu, lane < cluster ? x : 0);
      const int b = __reduce_add_sync(0xffffffffu, lane < part ? x : 0);
      if (m <= p) {
        left = m < p ? m : -1;
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
    for (int i = 0; i < kPer; ++i) count[i] = 0;
    for (int p = 0; p < cluster; ++p) {
      const int* from = peer(p)->hist[turn & 1];
#pragma unroll
      for (int i = 0; i < kPer; ++i) count[i] += from[kBins - 1 - (tid * kPer + i)];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
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
    const int bin = sm.pick[0], inside = sm.pick[2];
    need = sm.pick[1];
    low += (uint32_t)bin << shift;
    if (need == inside) {  // the whole interval stays
      top = low;
      left = -1;
      break;
    }
    if (shift == 0) {
      top = low;
      left = need;
      equal_before = __reduce_add_sync(0xffffffffu, lane < part ? peer(other)->hist[turn & 1][bin] : 0);
      break;
    }
    const uint32_t width = 1u << shift;
    if (inside <= kGather) {
      for (int t = tid; t < len; t += NT) {
        const uint32_t x = s_rank[t];
        if (x != kProtected && x >= low && x - low < width) sm.cand[atomicAdd(&sm.n_cand, 1)] = x - low;
      }
      sync_all();
      if (warp == 0) {
        int at = 0, at_mine = 0;
        for (int p = 0; p < cluster; ++p) {
          const Shared* of = peer(p);
          const int k = of->n_cand;
          if (p == part) at_mine = at;
          for (int i = lane; i < k; i += 32) sm.found[at + i] = of->cand[i];
          at += k;
        }
        __syncwarp();
        uint32_t v[kGather / 32];
#pragma unroll
        for (int i = 0; i < kGather / 32; ++i) v[i] = i * 32 + lane < at ? sm.found[i * 32 + lane] : 0;
        auto at_least = [&](uint32_t x) {
          int c = 0;
#pragma unroll
          for (int i = 0; i < kGather / 32; ++i) c += i * 32 + lane < at && v[i] >= x;
          return (int)__reduce_add_sync(0xffffffffu, c);
        };
        uint32_t x = 0;  // the need-th largest, relative to the interval
        for (int bit = shift - 1; bit >= 0; --bit)
          if (at_least(x | 1u << bit) >= need) x |= 1u << bit;
        int over = 0, equal = 0, ahead = 0;
#pragma unroll
        for (int i = 0; i < kGather / 32; ++i) {
          if (i * 32 + lane >= at) continue;
          over += v[i] > x;
          equal += v[i] == x;
          ahead += v[i] == x && i * 32 + lane < at_mine;
        }
        over = __reduce_add_sync(0xffffffffu, over);
        equal = __reduce_add_sync(0xffffffffu, equal);
        ahead = __reduce_add_sync(0xffffffffu, ahead);
        if (lane == 0) {
          sm.pick[0] = (int)(low + x);
          sm.pick[1] = equal == need - over ? -1 : need - over;
          sm.pick[2] = ahead;
        }
      }
      __syncthreads();
      top = (uint32_t)sm.pick[0];
      left = sm.pick[1];
      equal_before = sm.pick[2];
      break;
    }
    shift = max(0, shift - 10);
    int* next = sm.hist[(turn + 1) & 1];
    for (int t = tid; t < len; t += NT) {
      const uint32_t x = s_rank[t];
      if (x != kProtected && x >= low && x - low < width) atomicAdd(&next[(x - low) >> shift], 1);
    }
  }

  // 3. What is kept, a bit per slot ...
  const int words = (len + 31) / 32;
#pragma unroll 4
  for (int i = warp; i < words; i += kWarps) {
    const int t = i * 32 + lane;
    const uint32_t x = t < len ? s_rank[t] : 0;
    const uint32_t k = __ballot_sync(0xffffffffu, t < len && m > 0 && (left < 0 ? x >= top : x > top));
    const uint32_t q = __ballot_sync(0xffffffffu, t < len && x == top);
    if (lane == 0) s_kept[i] = k, s_equal[i] = q;
  }
  __syncthreads();
  const int each = (words + NT - 1) / NT;  // neighbouring words of a thread
  const int i0 = min(tid * each, words), i1 = min(i0 + each, words);
  if (left >= 0) {
    int eq = 0, total;
    for (int i = i0; i < i1; ++i) eq += __popc(s_equal[i]);
    int seen = equal_before + block_scan(eq, sm.warp_a, kWarps, &total);
    for (int i = i0; i < i1; ++i) {
      uint32_t q = s_equal[i], k = s_kept[i];
      const int here = __popc(q);
      if (seen + here <= left) {
        k |= q;
      } else {
        for (int j = seen; j < left; ++j) {  // the lowest left - seen of them
          k |= q & -q;
          q &= q - 1;
        }
      }
      seen += here;
      s_kept[i] = k;
    }
  }
  // ... and the row's lists.
  int counts = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t under = bits_below(lo + 32 * i, m), valid = bits_below(32 * i, len);
    counts += __popc(~s_kept[i] & under & valid) + (__popc(s_kept[i] & ~under) << 16);
  }
  int block_counts;
  const int before = block_scan(counts, sm.warp_a, kWarps, &block_counts);
  if (tid == 0) sm.counts = block_counts;
  sync_all();
  const int theirs = peer(other)->counts;
  int hole_at = (before & 0xFFFF) + (int)__reduce_add_sync(0xffffffffu, lane < part ? theirs & 0xFFFF : 0);
  int move_at = (int)((uint32_t)before >> 16) +
                (int)__reduce_add_sync(0xffffffffu, lane < part ? (int)((uint32_t)theirs >> 16) : 0);
  const int moves = (int)__reduce_add_sync(0xffffffffu, lane < cluster ? (int)((uint32_t)theirs >> 16) : 0);
  int32_t* empties = a.lists + (size_t)r * 2 * a.list_ld;
  int32_t* movers = empties + a.list_ld;
  for (int i = i0; i < i1; ++i) {
    const uint32_t under = bits_below(lo + 32 * i, m), valid = bits_below(32 * i, len);
    for (uint32_t x = ~s_kept[i] & under & valid; x; x &= x - 1) empties[hole_at++] = lo + 32 * i + __ffs(x) - 1;
    for (uint32_t x = s_kept[i] & ~under; x; x &= x - 1) movers[move_at++] = lo + 32 * i + __ffs(x) - 1;
  }
  // What stays in place, and the slots beyond m that nothing moves from (the others are
  // read once more by their move, which empties them).
#pragma unroll 4
  for (int t = tid; t < len; t += NT) {
    const bool kept = s_kept[t >> 5] >> (t & 31) & 1;
    if (lo + t < m) {
      if (kept && w_out != w) w_out[t] = w[t];
      if (kept && pos_out != pos) pos_out[t] = pos[t];
    } else if (!kept) {
      w_out[t] = 0.f;
      pos_out[t] = -1;
    }
  }
  if (part == 0 && tid == 0) {
    a.ctx_out[r] = m;  // every block has read its length
    a.counts[r] = moves;
  }
  if (cluster > 1) all.sync();  // no block leaves while another may read its counts
}

// Moves [128 i, 128 (i + 1)) of one row.  A thread each looks the pages up and moves weight
// and position; then D / 16 lanes a key copy the codes, 16 bytes a lane, 4 keys at once.
constexpr int kMoveThreads = 256;
constexpr int kMoves = 128;

template <int W>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(Args a, int blocks_per_row) {
  constexpr int G = 2 * W;
  constexpr int kGroups = kMoveThreads / G;
  constexpr int kFlight = 4;
  __shared__ uint32_t s_from[kMoves], s_to[kMoves];
  const int tid = threadIdx.x;
  const int r = blockIdx.x / blocks_per_row;
  const int first = (blockIdx.x - r * blocks_per_row) * kMoves;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int count = min(__ldcg(a.counts + r) - first, kMoves);
  if (count <= 0) return;
  if (tid < count) {
    const int32_t* empties = a.lists + (size_t)r * 2 * a.list_ld + first;
    const int dst = __ldcg(empties + tid), src = __ldcg(empties + a.list_ld + tid);
    const long long from = a.pages.slot(r, src), to = a.pages.slot(r, dst);
    const bool ok = from >= 0 && to >= 0;
    if (!ok) raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
    s_from[tid] = ok ? (uint32_t)from : 0xffffffffu;
    s_to[tid] = (uint32_t)to;
    const long long row = r * a.ld;
    const float w = a.w_in[row + src];
    const int32_t p = a.pos_in[row + src];
    a.w_out[row + dst] = w;
    a.pos_out[row + dst] = p;
    a.w_out[row + src] = 0.f;
    a.pos_out[row + src] = -1;
    if (ok && a.v_scale) a.v_scale[to] = a.v_scale[from];
  }
  __syncthreads();
  const int sub = tid % G, group = tid / G;
  const bool words = sub < W / 4;
  for (int i0 = group; i0 < count; i0 += kGroups * kFlight) {
    uint4 v[kFlight], k[kFlight];
    uint32_t from[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int i = i0 + u * kGroups;
      from[u] = i < count ? s_from[i] : 0xffffffffu;
      if (from[u] == 0xffffffffu) continue;
      v[u] = *(reinterpret_cast<const uint4*>(a.v) + (size_t)from[u] * G + sub);
      if (words) k[u] = *(reinterpret_cast<const uint4*>(a.k) + (size_t)from[u] * (W / 4) + sub);
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if (from[u] == 0xffffffffu) continue;
      const size_t to = s_to[i0 + u * kGroups];
      *(reinterpret_cast<uint4*>(a.v) + to * G + sub) = v[u];
      if (words) *(reinterpret_cast<uint4*>(a.k) + to * (W / 4) + sub) = k[u];
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

// Lists first, then the counts.
inline size_t lists_bytes(long long n_kv, long long cap) { return (size_t)n_kv * 2 * list_ld(cap) * sizeof(int32_t); }
inline size_t scratch_bytes(long long n_kv, long long cap) { return lists_bytes(n_kv, cap) + (size_t)n_kv * sizeof(int32_t); }

constexpr size_t kMaxSmem = 227 * 1024;
constexpr int kBlockKeys = 16384;  // of a row per block, while 16 blocks do

inline cudaError_t setup() {
  cudaError_t e = cudaSuccess;
  auto set = [&](const void* kernel) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  };
  set(reinterpret_cast<const void*>(select_kernel<512, 4>));
  set(reinterpret_cast<const void*>(select_kernel<1024, 2>));
  return e;
}

inline cudaError_t launch(const Args& a, int n_sm, cudaStream_t st) {
  const long long cap = (long long)a.pages.num_blocks * a.pages.block_size;
  int cluster = 1;
  auto part = [&](int c) { return ((cap + c - 1) / c + 31) / 32 * 32; };
  while (cluster < kMaxCluster && part(cluster) > kBlockKeys) cluster *= 2;
  // Few rows: more blocks a row while the device has room and a block keeps 4096 keys.
  while (cluster < 8 && (long long)a.n_kv * cluster * 2 <= n_sm && part(cluster) >= 8192) cluster *= 2;
  const long long keys = part(cluster);
  const size_t smem = sizeof(Shared) + (size_t)keys * 4 + (size_t)keys / 32 * 8;
  if (smem > kMaxSmem) {
    evict_long_kernel<<<(unsigned)a.n_kv, kLongThreads, 0, st>>>(a);
    return cudaGetLastError();
  }
  const int threads = keys > 8192 ? 1024 : 512;
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
  cudaError_t e = threads == 1024 ? cudaLaunchKernelEx(&cfg, select_kernel<1024, 2>, a, cluster, (int)keys)
                                  : cudaLaunchKernelEx(&cfg, select_kernel<512, 4>, a, cluster, (int)keys);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // The most moves a row can have: its budget, or what lies beyond it.
  const long long most = a.keep_rows ? cap / 2 : std::min<long long>(a.keep, cap - a.keep);
  if (most <= 0) return cudaSuccess;
  const int per_row = (int)((most + kMoves - 1) / kMoves);
  cudaLaunchConfig_t move = {};
  move.gridDim = dim3((unsigned)((long long)a.n_kv * per_row));
  move.blockDim = dim3(kMoveThreads);
  move.stream = st;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  move.attrs = pdl;
  move.numAttrs = 1;
  e = a.row_words == 8 ? cudaLaunchKernelEx(&move, move_kernel<8>, a, per_row)
                       : cudaLaunchKernelEx(&move, move_kernel<4>, a, per_row);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace evict
}  // namespace hyp
