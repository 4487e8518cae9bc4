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
  const uint32_t b = __float_as_uint(w + 0.f);
  const uint32_t x = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return w != w ? 0 : x;
}

// ---------------------------------------------------------------------------
// select_kernel: a cluster of up to 16 blocks per row, each with its part of the row's
// ranks in shared memory.
//
//   1. Read weights and positions once; the row's newest position and the range of its
//      ranks by way of distributed shared memory.
//   2. The m-th largest rank, by histograms of kBins equal intervals of the range that is
//      left (12 bits a turn), until an interval is kept whole or holds at most kGather
//      ranks: those are gathered and each is counted against the others.  Sums of attention
//      weights take one turn, now and then two.  So many intervals also keep the lanes of a
//      warp from adding to the same one: with 1024, 4 to 5 of 32 met.
//   3. A bit per slot says what is kept.  The counts of 32 slots are added up per word, and
//      each warp writes its slots' places into the row's two lists (slots that empty below
//      m, keys that move), in slot order.
//
// move_kernel: the moves of all rows, 128 a block (64 at head_dim 256), whichever row they
// belong to.
//
// 128 rows of 32768 keys cut to 4096: selection 35 us, 34 MB of sums and positions, bound by
// its instructions (54 % of the issue slots) and barriers; moves 31 us, scattered rows of 128,
// 16 and 4 bytes, 147 MB of DRAM traffic at 4.5 TB/s.  Both in one kernel: 158 us, since a
// row's moves are then one SM's.  512 rows of 4097 cut to 4096: 25 us.  The instances of 512
// and 1024 threads are held to 32 registers for their blocks an SM and spill (104 and 44
// bytes of stores a thread).
// ---------------------------------------------------------------------------
constexpr int kBins = 4096;  // two 16-bit counts a word: a block has at most 52k keys
constexpr int kBinBits = 12;
constexpr int kGather = 256;
constexpr int kMaxCluster = 16;

struct __align__(16) Shared {
  uint32_t hist[2][kBins / 2];
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

// One more in interval `bin`.
__device__ __forceinline__ void count_one(uint32_t* hist, uint32_t bin) { atomicAdd(hist + (bin >> 1), 1u << (16 * (bin & 1))); }

// Bits of word `at` (slots at .. at + 31) that lie below `end`.
__device__ __forceinline__ uint32_t bits_below(int at, int end) {
  const int k = end - at;
  return k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1u;
}

// Four neighbouring values, `n` of them real; one read or write where `vec`.
template <typename V, typename T>
__device__ __forceinline__ void load4(T (&x)[4], const T* p, int n, bool vec) {
  if (vec && n >= 4) {
    const V v = *reinterpret_cast<const V*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = j < n ? p[j] : T(0);
  }
}
template <typename V, typename T>
__device__ __forceinline__ void store4(T* p, const T (&x)[4], int n, bool vec) {
  if (vec && n >= 4) {
    V v;
    v.x = x[0], v.y = x[1], v.z = x[2], v.w = x[3];
    *reinterpret_cast<V*>(p) = v;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[j] = x[j];
  }
}

// Each thread works on 4 neighbouring slots at a time; `vec`: the rows lie on 16 bytes.
template <int NT, int kBlocks>
__global__ void __launch_bounds__(NT, kBlocks) select_kernel(Args a, int cluster, int keys, bool vec, bool move_here) {
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
#pragma unroll 2
  for (int t = 4 * tid; t < len; t += 4 * NT) {
    const int real = len - t;
    float wv[4];
    int32_t pv[4];
    uint32_t x[4];
    load4<float4>(wv, w + t, real, vec);
    load4<int4>(pv, pos + t, real, vec);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = rank_of(wv[j]);
      if (j < real) {
        newest = max(newest, pv[j]);
        low = min(low, x[j]);
        high = max(high, x[j]);
      }
    }
    *reinterpret_cast<uint4*>(s_rank + t) = make_uint4(x[0], x[1], x[2], x[3]);
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) sm.warp_a[warp] = newest, sm.warp_lo[warp] = low, sm.warp_hi[warp] = high;
  for (int i = tid; i < kBins / 8; i += NT) reinterpret_cast<uint4*>(sm.hist[0])[i] = make_uint4(0, 0, 0, 0);
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
  int shift = max(0, 32 - __clz(high - low) - kBinBits);
  int mine = 0;
#pragma unroll 2
  for (int t = 4 * tid; t < len; t += 4 * NT) {
    const int real = len - t;
    int32_t pv[4];
    load4<int4>(pv, pos + t, real, vec);
    const uint4 v = *reinterpret_cast<const uint4*>(s_rank + t);
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= real) continue;
      // newest - p may pass 2^31, not 2^32
      if (pv[j] < a.sink || (uint32_t)newest - (uint32_t)pv[j] < (uint32_t)a.recent) {
        s_rank[t + j] = kProtected;
        ++mine;
      } else {
        count_one(sm.hist[0], (x[j] - low) >> shift);
      }
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
    }
    // This thread's intervals, kPer neighbours; thread 0 has the highest.
    constexpr int kPer = kBins / NT;
    static_assert(kPer >= 4, "a thread reads its intervals 4 at a time");
    const int bin0 = kBins - kPer * (tid + 1);
    int count[kPer] = {}, sum = 0;
    for (int p = 0; p < cluster; ++p) {
      const uint32_t* from = peer(p)->hist[turn & 1] + bin0 / 2;
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        const uint2 x = *reinterpret_cast<const uint2*>(from + i / 2);
        count[i] += x.x & 0xFFFF, count[i + 1] += x.x >> 16;
        count[i + 2] += x.y & 0xFFFF, count[i + 3] += x.y >> 16;
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += count[i];
    int total;
    int above = block_scan(sum, sm.warp_a, kWarps, &total);
    if (above < need && need <= above + sum) {
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i) {
        if (above < need && need <= above + count[i]) {
          sm.pick[0] = bin0 + i;
          sm.pick[1] = need - above;
          sm.pick[2] = count[i];
        }
        above += count[i];
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
      equal_before = __reduce_add_sync(0xffffffffu, lane < part ? (int)(peer(other)->hist[turn & 1][bin >> 1] >> (16 * (bin & 1)) & 0xFFFF) : 0);
      break;
    }
    const uint32_t width = 1u << shift;
    if (inside <= kGather) {
      for (int t = 4 * tid; t < len; t += 4 * NT) {
        const uint4 v = *reinterpret_cast<const uint4*>(s_rank + t);
        const uint32_t x[4] = {v.x - low, v.y - low, v.z - low, v.w - low};
        if (min(min(x[0], x[1]), min(x[2], x[3])) >= width) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (t + j < len && x[j] < width && x[j] + low != kProtected) sm.cand[atomicAdd(&sm.n_cand, 1)] = x[j];
      }
      sync_all();
      // All blocks' candidates, in the order of the blocks, padded with zeros; a thread
      // counts one of them.
      int at = 0, ahead_end = 0;
      for (int p = 0; p < cluster; ++p) {
        const Shared* of = peer(p);
        const int k = of->n_cand;
        if (p == part) ahead_end = at;
        if (tid < k) sm.found[at + tid] = of->cand[tid];
        at += k;
      }
      if (tid < 4 && at + tid < kGather) sm.found[at + tid] = 0;
      __syncthreads();
      const uint32_t x = tid < at ? sm.found[tid] : 0;
      const uint32_t first = sm.found[0];
      if (__syncthreads_and(tid >= at || x == first)) {  // keys that nothing has looked at share a sum
        if (tid == 0) sm.pick[0] = (int)first, sm.pick[1] = need;
      } else if (warp * 32 < at) {
        int over = 0, not_under = 0;
#pragma unroll 4
        for (int i = 0; i < (at + 3) / 4; ++i) {
          const uint4 y = reinterpret_cast<const uint4*>(sm.found)[i];
          over += (y.x > x) + (y.y > x) + (y.z > x) + (y.w > x);
          not_under += (y.x >= x) + (y.y >= x) + (y.z >= x) + (y.w >= x);
        }
        if (x == 0) not_under = at;
        if (tid < at && over < need && need <= not_under) {  // all such threads hold the same rank
          sm.pick[0] = (int)x;
          sm.pick[1] = need == not_under ? -1 : need - over;
        }
      }
      __syncthreads();
      const uint32_t found = (uint32_t)sm.pick[0];
      left = sm.pick[1];
      equal_before = __syncthreads_count(tid < ahead_end && x == found);
      top = low + found;
      break;
    }
    shift = max(0, shift - kBinBits);
    // The other buffer's readers, in the turn before, are past this turn's sync.
    uint32_t* next = sm.hist[(turn + 1) & 1];
    for (int i = tid; i < kBins / 8; i += NT) reinterpret_cast<uint4*>(next)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int t = tid; t < len; t += NT) {
      const uint32_t x = s_rank[t];
      if (x != kProtected && x >= low && x - low < width) count_one(next, (x - low) >> shift);
    }
  }

  // 3. What is kept, a bit per slot ...
  const int words = (len + 31) / 32;
  for (int t0 = 128 * warp; t0 < len; t0 += 4 * NT) {  // a warp: 4 words
    const int t = t0 + 4 * lane, real = len - t;
    const uint4 v = *reinterpret_cast<const uint4*>(s_rank + min(t, keys - 4));
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
    uint32_t k = 0, q = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      k |= (j < real && (left < 0 ? x[j] >= top : x[j] > top)) << j;
      q |= (j < real && x[j] == top) << j;
    }
    k <<= 4 * (lane & 7), q <<= 4 * (lane & 7);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) k |= __shfl_xor_sync(0xffffffffu, k, o);
    if (left >= 0) {
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) q |= __shfl_xor_sync(0xffffffffu, q, o);
    }
    if ((lane & 7) == 0 && real > 0) s_kept[t >> 5] = m > 0 ? k : 0, s_equal[t >> 5] = q;
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
  // ... and the row's lists: slots that empty | keys that move << 16, before each word.
  int counts = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t under = bits_below(lo + 32 * i, m), valid = bits_below(32 * i, len);
    counts += __popc(~s_kept[i] & under & valid) + (__popc(s_kept[i] & ~under) << 16);
  }
  int block_counts;
  int before = block_scan(counts, sm.warp_a, kWarps, &block_counts);
  for (int i = i0; i < i1; ++i) {
    const uint32_t under = bits_below(lo + 32 * i, m), valid = bits_below(32 * i, len);
    s_equal[i] = (uint32_t)before;  // the ties are settled
    before += __popc(~s_kept[i] & under & valid) + (__popc(s_kept[i] & ~under) << 16);
  }
  if (tid == 0) sm.counts = block_counts;
  sync_all();
  const uint32_t theirs = (uint32_t)peer(other)->counts;
  const int hole_at = (int)__reduce_add_sync(0xffffffffu, lane < part ? theirs & 0xFFFF : 0);
  const int move_at = (int)__reduce_add_sync(0xffffffffu, lane < part ? theirs >> 16 : 0);
  const int moves = (int)__reduce_add_sync(0xffffffffu, lane < cluster ? theirs >> 16 : 0);
  int32_t* empties = a.lists + (size_t)r * 2 * a.list_ld + hole_at;
  int32_t* movers = a.lists + ((size_t)r * 2 + 1) * a.list_ld + move_at;
  // Into other tensors, what stays is copied and all beyond m emptied; in place, what
  // moves is still to be read, so its move empties it.  A slot that empties gets its key's
  // values from the move.
  const bool w_else = w_out != w, pos_else = pos_out != pos;
  const int split = min(max(m - lo, 0), len);  // this block's slots below m
  for (int t = 4 * tid; t < split; t += 4 * NT) {
    const int real = split - t, bit0 = t & 31;
    if (w_else) {
      float x[4];
      load4<float4>(x, w + t, real, vec);
      store4<float4>(w_out + t, x, real, vec);
    }
    if (pos_else) {
      int32_t x[4];
      load4<int4>(x, pos + t, real, vec);
      store4<int4>(pos_out + t, x, real, vec);
    }
    const uint32_t gone = ~s_kept[t >> 5] & bits_below(t - bit0, split);
    uint32_t here = gone >> bit0 & 0xF;
    if (here) {
      int32_t* to = empties + (s_equal[t >> 5] & 0xFFFF) + __popc(gone & ((1u << bit0) - 1u));
      for (; here; here &= here - 1) *to++ = lo + t + __ffs(here) - 1;
    }
  }
  for (int t = (split & ~3) + 4 * tid; t < len; t += 4 * NT) {
    const int bit0 = t & 31;
    const uint32_t stay = s_kept[t >> 5] & ~bits_below(t - bit0, split);
    uint32_t here = stay >> bit0 & 0xF;
    if (t >= split && (here == 0 || (w_else && pos_else))) {
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      const int32_t none[4] = {-1, -1, -1, -1};
      store4<float4>(w_out + t, zero, len - t, vec);
      store4<int4>(pos_out + t, none, len - t, vec);
    } else {
#pragma unroll 1
      for (int j = max(split - t, 0); j < min(len - t, 4); ++j) {
        const bool moves_on = here >> j & 1;
        if (w_else || !moves_on) w_out[t + j] = 0.f;
        if (pos_else || !moves_on) pos_out[t + j] = -1;
      }
    }
    if (here) {
      int32_t* to = movers + (s_equal[t >> 5] >> 16) + __popc(stay & ((1u << bit0) - 1u));
      for (; here; here &= here - 1) *to++ = lo + t + __ffs(here) - 1;
    }
  }
  if (part == 0 && tid == 0) {
    a.ctx_out[r] = m;  // every block has read its length
    a.counts[r] = moves;
  }
  if (cluster > 1) all.sync();  // no block leaves while another may read its counts
  if (!move_here) return;
  // A few moves (a step over the budget makes one): here, without a launch of their own.
  __syncthreads();
  const int W = a.row_words, G = 2 * W, sub = tid % G;
  const long long row = r * a.ld;
  for (int i = tid / G; i < moves; i += NT / G) {
    const int dst = __ldcg(empties + i), src = __ldcg(movers + i);
    const long long from = a.pages.slot(r, src), to = a.pages.slot(r, dst);
    if (sub == 0) {
      const float wv = a.w_in[row + src];
      const int32_t pv = a.pos_in[row + src];
      a.w_out[row + dst] = wv;
      a.pos_out[row + dst] = pv;
      if (a.w_out == a.w_in) a.w_out[row + src] = 0.f;
      if (a.pos_out == a.pos_in) a.pos_out[row + src] = -1;
    }
    if (from < 0 || to < 0) {
      if (sub == 0) raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
      continue;
    }
    reinterpret_cast<uint4*>(a.v)[to * G + sub] = reinterpret_cast<const uint4*>(a.v)[from * G + sub];
    if (sub < W / 4) reinterpret_cast<uint4*>(a.k)[to * (W / 4) + sub] = reinterpret_cast<const uint4*>(a.k)[from * (W / 4) + sub];
    if (sub == 0 && a.v_scale) a.v_scale[to] = a.v_scale[from];
  }
}

// Moves [kMoves i, kMoves (i + 1)) of one row.  A thread looks a move's pages up; D / 16
// lanes copy a key's codes, 16 bytes each and kFlight keys at once; and while those are
// under way a thread each takes a move's words, weight, position and slot scale, whose
// destinations lie side by side.
constexpr int kMoveThreads = 256;
constexpr int kFlight = 4;

template <int W>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(Args a, int blocks_per_row) {
  constexpr int G = 2 * W;
  constexpr int kGroups = kMoveThreads / G;
  constexpr int kMoves = kGroups * kFlight;
  constexpr uint32_t kNoRow = 0xffffffffu;
  __shared__ uint32_t s_from[kMoves], s_to[kMoves];
  const int tid = threadIdx.x, sub = tid % G, group = tid / G;
  const int r = blockIdx.x / blocks_per_row;
  const int first = (blockIdx.x - r * blocks_per_row) * kMoves;
  const int32_t* empties = a.lists + (size_t)r * 2 * a.list_ld;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int count = min(__ldcg(a.counts + r) - first, kMoves);
  if (count <= 0) return;
  int src = 0, dst = 0;
  uint32_t from = kNoRow, to = kNoRow;
  if (tid < count) {
    dst = __ldcg(empties + first + tid);
    src = __ldcg(empties + a.list_ld + first + tid);
    from = (uint32_t)a.pages.slot(r, src);
    to = (uint32_t)a.pages.slot(r, dst);
    if (from == kNoRow || to == kNoRow) {
      raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
      from = kNoRow;
    }
  }
  if (tid < kMoves) s_from[tid] = from, s_to[tid] = to;
  __syncthreads();
  uint4 v[kFlight];
  uint32_t at[kFlight];
#pragma unroll
  for (int u = 0; u < kFlight; ++u) {
    at[u] = s_from[u * kGroups + group];
    if (at[u] != kNoRow) v[u] = *(reinterpret_cast<const uint4*>(a.v) + (size_t)at[u] * G + sub);
  }
  if (tid < count) {
    const long long row = r * a.ld;
    const float w = a.w_in[row + src];
    const int32_t p = a.pos_in[row + src];
    if (from != kNoRow) {
      uint4 k[W / 4];
#pragma unroll
      for (int i = 0; i < W / 4; ++i) k[i] = *(reinterpret_cast<const uint4*>(a.k) + (size_t)from * (W / 4) + i);
      const float scale = a.v_scale ? a.v_scale[from] : 0.f;
#pragma unroll
      for (int i = 0; i < W / 4; ++i) *(reinterpret_cast<uint4*>(a.k) + (size_t)to * (W / 4) + i) = k[i];
      if (a.v_scale) a.v_scale[to] = scale;
    }
    a.w_out[row + dst] = w;
    a.pos_out[row + dst] = p;
    if (a.w_out == a.w_in) a.w_out[row + src] = 0.f;
    if (a.pos_out == a.pos_in) a.pos_out[row + src] = -1;
  }
#pragma unroll
  for (int u = 0; u < kFlight; ++u)
    if (at[u] != kNoRow) *(reinterpret_cast<uint4*>(a.v) + (size_t)s_to[u * kGroups + group] * G + sub) = v[u];
}

// ---------------------------------------------------------------------------
// Rows too long for 16 blocks' shared memory (from about 800,000 keys): one block a row, which
// reads the ranks anew for each turn.  8 rows of 131072, which do not need it: 1137 us, the
// clusters 46.  8 rows of 820,032: 6.6 ms, where clusters take 0.16 for rows of 803,200.
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
// Moves of a row at most, that the selection makes itself: no launch of their own, but one
// block's.  512 rows cut to 4096 by 1 key: 20.2 us here, 21.3 by move_kernel; by 64: 22.6 both;
// by 128: 25.7 and 23.9; by 512: 53 and 39.  64 rows: 13.4 and 14.4, 14.6 and 14.8, 17.2 and
// 14.7, 28 and 14.
constexpr int kMovesHere = 128;
constexpr int kBlockKeys = 16384;  // of a row per block, while 16 blocks do

inline cudaError_t setup() {
  cudaError_t e = cudaSuccess;
  auto set = [&](const void* kernel) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  };
  set(reinterpret_cast<const void*>(select_kernel<256, 4>));
  set(reinterpret_cast<const void*>(select_kernel<512, 4>));
  set(reinterpret_cast<const void*>(select_kernel<1024, 2>));
  return e;
}

inline cudaError_t launch(const Args& a, int n_sm, cudaStream_t st) {
  const long long cap = (long long)a.pages.num_blocks * a.pages.block_size;
  int cluster = 1;
  auto part = [&](int c) { return ((cap + c - 1) / c + 31) / 32 * 32; };
  while (cluster < kMaxCluster && part(cluster) > kBlockKeys) cluster *= 2;
  // Few rows: more blocks a row while the device has room and a block keeps 4096 keys.  Not 16:
  // 8 rows of 131072 take 89 us with clusters of 16, 36 with 8; 4 rows 59 and 34.
  while (cluster < 8 && (long long)a.n_kv * cluster * 2 <= n_sm && part(cluster) >= 8192) cluster *= 2;
  const long long keys = part(cluster);
  const size_t smem = sizeof(Shared) + (size_t)keys * 4 + (size_t)keys / 32 * 8;
  if (smem > kMaxSmem) {
    evict_long_kernel<<<(unsigned)a.n_kv, kLongThreads, 0, st>>>(a);
    return cudaGetLastError();
  }
  // Threads by the keys of a block.  Rows that fill the device, cut by one key and to a quarter,
  // us with 256 / 512 / 1024 threads: 2049 keys 25 / 28 / 44 and 53 / 57 / 68, 4097 20 / 23 / 34
  // and 47 / 49 / 60, 5001 22.7 / 23.6 / 31 and 48 / 48 / 57, 6001 26.1 / 25.7 / 34 and
  // 51 / 49 / 57, 8192 27 / 23 / 26 and 60 / 57 / 51, 12289 36 / 30 / 33 and 68 / 63 / 56,
  // 16384 40 / 28 / 24 and 64 / 53 / 51: 512 overtake 256 between 5000 and 6000 keys, 1024
  // overtake 512 from 8192 on, first where many keys go.
  const int threads = keys > 8192 ? 1024 : keys > 4608 ? 512 : 256;
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
  auto on16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool vec = a.ld % 4 == 0 && on16(a.w_in) && on16(a.w_out) && on16(a.pos_in) && on16(a.pos_out);
  auto kernel = threads == 1024 ? select_kernel<1024, 2> : threads == 512 ? select_kernel<512, 4> : select_kernel<256, 4>;
  // The most moves a row can have: its budget, or what lies beyond it.
  const long long most = a.keep_rows ? cap / 2 : std::min<long long>(a.keep, cap - a.keep);
  const bool move_here = cluster == 1 && most <= kMovesHere;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, cluster, (int)keys, vec, move_here);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess || move_here || most <= 0) return e;
  const int moves = kMoveThreads / (2 * a.row_words) * kFlight;  // of a block
  const int per_row = (int)((most + moves - 1) / moves);
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
