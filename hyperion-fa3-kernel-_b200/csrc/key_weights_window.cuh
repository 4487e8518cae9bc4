// key_weights_window.cuh -- key_weights.cuh for windows of many query rows: the scores on the
// tensor core.
//
// Two kernels over the same tiles.  A block takes up to 256 query rows of one KV row, kept in
// shared memory as e4m3 +-1 bytes for the whole call, and streams a chunk of the row's keys
// past them, 128 at a time.  Each tile of 128 queries x 128 keys is D / 32 tcgen05.mma of
// kind::f8f6f4: the products of +-1 sum to D - 2 popcount(q ^ k) exactly in the f32
// accumulator.
//
//   kSum false   rows of the accumulator are queries, columns keys: each thread sums E over
//                its query's keys, for the softmax denominators;
//   kSum true    rows are keys, columns queries (the two operands change places): each
//                thread sums E / l over the queries, for the key's weight.
//
// Here E = exp(inv_sqrt_d s), relative to a score of 0: within kFlat's bound it stays between
// e^-40 and e^40, and typical exponents are small, so their rounding is too.  It is computed
// in two ways side by side, because either alone would hold the kernel up.  Some columns
// take 2^x on the exponential unit (a warp instruction every 2 cycles of an SM); the others
// read a table in shared memory (one every cycle, beside the 1 / l of each column, which
// costs as much again).  The table's address is one FMA away: in units of the smallest f32,
// 2^-149, a subnormal number's bits are its value, so s times -2, plus 2 D and the table's
// address, is the address of E[p] exactly.
//
// The two accumulators of a key tile (128 columns each, two blocks on an SM) are computed
// and read in turn: while the threads read one, the tensor core fills the other, and the
// next tile's sign bits, loaded at the start of a turn, are expanded at its end.
//
// 32 rows of 256 queries and up to 16384 keys of 128 dims: 90 us for both kernels, where the
// products alone would take 15 at the bf16 rate and the bytes 1.5.  What bounds them is the
// exponentials (the table alone 97 us, the unit alone 119), a block's setup (40 % of its time
// at 4 tiles a chunk; 8 tiles leave SMs without work) and 16 warps an SM.  512 threads a
// block, one on an SM: 122 us.
//
// Every tile of a row is computed for every group, also where causal queries see none of it:
// whole prompts (4 sequences of 8 KV heads, 4 query heads each) 0.23 ms at 1024 rows, 0.58 at
// 2048, 2.2 at 4096; without the mask 0.18, 0.46 and 1.8.  Fewer query rows than 128 leave
// columns that hold no query but are computed: 64 rows of 8192 keys with 32 queries 69 us, with
// 16, by the popcount kernels, 22.
#pragma once

#include "key_weights.cuh"
#include "tile_kernel.cuh"

namespace hyp {
namespace kweights {

constexpr int kWinQueries = 256;  // of a block
constexpr int kWinKeys = 128;     // of a tile
constexpr int kWinThreads = 256;
constexpr uint32_t kWinTmemCols = 256;

struct WindowArgs {
  int groups;   // of kWinQueries queries
  int chunks;   // per row
  int tiles;    // of a chunk
  float* part;  // [n_kv, chunks, groups * kWinQueries]: sums of E
};

template <int D>
struct WindowSmem {
  alignas(1024) uint8_t q[2][D / 128][128 * 128];
  alignas(1024) uint8_t k[2][D / 128][128 * 128];
  float e[D + 4];
  alignas(16) uint16_t mask[2][8];  // keys of each tile that exist
  int end[kWinQueries];             // keys each query sees, INT_MAX for a place without a query
  alignas(16) float inv[kWinQueries];  // 1 / l, 0 for a place without a query
  float half[2][128];               // sums of the upper 64 columns
  float out[kWinThreads * 8];       // the chunk's key sums (at most 16 tiles)
  int min_end;
  alignas(8) uint64_t ready[2], drain;
  uint32_t tmem_base;
  WaitCtl ctl;
};

constexpr int kMaxChunkTiles = 16;

// Sign words of half a row (16 bytes at head_dim 256, 8 at 128).
template <int D>
struct HalfRow {
  uint32_t w[D / 64];
};

template <int D>
__device__ __forceinline__ HalfRow<D> load_half(const uint32_t* row, int half) {
  HalfRow<D> h;
  if constexpr (D == 128) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(row) + half);
    h.w[0] = v.x, h.w[1] = v.y;
  } else {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row) + half);
    h.w[0] = v.x, h.w[1] = v.y, h.w[2] = v.z, h.w[3] = v.w;
  }
  return h;
}

// Half a row of +-1 bytes into a tile of 128-byte swizzled rows (one block of 128 dims, two
// at head_dim 256).
template <int D>
__device__ __forceinline__ void expand_half(const HalfRow<D>& h, uint32_t tile, int row, int half) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {  // 16 dims each
    const int chunk = half * (D / 32) + i;
    const uint32_t at = tile + (chunk / 8) * (128 * 128) + tile::sw128_off(row, chunk % 8);
    tile::st_shared_v4(at, tile::expand16((h.w[i / 2] >> (16 * (i & 1))) & 0xFFFFu));
  }
}

__device__ __forceinline__ float shared_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

constexpr uint32_t kUnitSum = 0x6D, kUnitL = 0x49;

// Sum over 64 accumulator columns of E (kSum: E / l of the column's query).  Masked: column i
// counts where bit i of `on` is set.
template <bool kSum, bool kMasked>
__device__ __forceinline__ float sum_columns(uint32_t s_col, float e_bias, float x_mul, const float* inv, uint64_t on) {
  // Of 8 column pairs, those that go to the exponential unit: 5 beside the reads of 1 / l, 3
  // without.
  constexpr uint32_t kUnit = kSum ? kUnitSum : kUnitL;
  const float kMinusTwo = __uint_as_float(0x80000002u);  // -2 x 2^-149
  float2 acc[2] = {};
  // 16 columns are read while the 16 before them are worked on (90.0 us against 91.5 for 32
  // read, waited for and used: 32 rows of 256 queries and up to 16384 keys).
  uint32_t v[2][16];
  tc::ld16(s_col, v[0]);
  tc::ld_wait_regs(v[0]);
#pragma unroll
  for (int cc = 0; cc < 64; cc += 16) {
    uint32_t(&now)[16] = v[cc / 16 & 1];
    if (cc < 48) tc::ld16(s_col + cc + 16, v[(cc / 16 + 1) & 1]);
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      float4 scale = make_float4(1.f, 1.f, 1.f, 1.f);
      if (kSum) scale = *reinterpret_cast<const float4*>(inv + cc + i);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float2 sc = make_float2(__uint_as_float(now[i + j]), __uint_as_float(now[i + j + 1]));
        float2 w;
        if (kUnit >> ((i + j) / 2 % 8) & 1) {
          const float2 x = __fmul2_rn(sc, make_float2(x_mul, x_mul));
          w = make_float2(ex2_approx(x.x), ex2_approx(x.y));
        } else {
          const float2 at = __ffma2_rn(sc, make_float2(kMinusTwo, kMinusTwo), make_float2(e_bias, e_bias));
          w = make_float2(shared_f32(__float_as_uint(at.x)), shared_f32(__float_as_uint(at.y)));
        }
        if (kMasked) {
          if (!(on >> (cc + i + j) & 1)) w.x = 0.f;
          if (!(on >> (cc + i + j + 1) & 1)) w.y = 0.f;
        }
        if (kSum) {
          acc[j / 2] = __ffma2_rn(w, j ? make_float2(scale.z, scale.w) : make_float2(scale.x, scale.y), acc[j / 2]);
        } else {
          acc[j / 2] = __fadd2_rn(acc[j / 2], w);
        }
      }
    }
    if (cc < 48) tc::ld_wait_regs(v[(cc / 16 + 1) & 1]);
  }
  const float2 all = __fadd2_rn(acc[0], acc[1]);
  return all.x + all.y;
}

template <int D, bool kSum>
__global__ void __launch_bounds__(kWinThreads, D == 128 ? 2 : 1) window_kernel(Args a, WindowArgs c) {
  constexpr int W = D / 32;
  extern __shared__ uint8_t raw[];
  auto& sm = *reinterpret_cast<WindowSmem<D>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // A block: (row, chunk) and, for the denominators, one group of queries.
  const int per_row = kSum ? c.chunks : c.chunks * c.groups;
  const int r = blockIdx.x / per_row;
  const int in_row = blockIdx.x - r * per_row;
  const int chunk = kSum ? in_row : in_row / c.groups;
  const int k0 = chunk * c.tiles * kWinKeys;
  const int n = a.pages.context(__ldg(a.ctx_lens + r), a.err, !kSum && in_row == 0 && tid == 0);
  if (k0 >= n) {
    if (kSum) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int k1 = min(k0 + c.tiles * kWinKeys, n);
  const int tiles = (k1 - k0 + kWinKeys - 1) / kWinKeys;
  const int rows = a.kv_group * a.n_q;

  if (tid == 0) {
    mbar_init(&sm.ready[0], 1);
    mbar_init(&sm.ready[1], 1);
    mbar_init(&sm.drain, 1);
    sm.ctl.flag = 0;
    sm.ctl.limit = a.wait_cycles;
    fence_mbar_init();
  }
  if (warp == 0) {
    tc::tmem_alloc(&sm.tmem_base, kWinTmemCols);
    tc::tmem_relinquish();
  }
  for (int j = tid; j <= D; j += kWinThreads) sm.e[j] = expf(a.inv_sqrt_d * (float)(D - 2 * j));
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = sm.tmem_base;
  // Only now that every block has its tensor memory: one of the next grid, which holds some
  // while it waits for this grid, can then not stand in the way of one of this.
  if (!kSum) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int row = tid >> 1, half = tid & 1;  // of the expansion
  const uint32_t q_tile = smem_u32(&sm.q[0][0][0]), k_tile = smem_u32(&sm.k[0][0][0]);
  constexpr uint32_t kTile = D / 128 * 128 * 128;
  const uint64_t q_desc = tc::sw128_desc(q_tile, 16, 1024), k_desc = tc::sw128_desc(k_tile, 16, 1024);
  // Thread 0, behind a barrier: accumulator s of the tile in key buffer `buf`, the block's
  // product `nth`.  The fence orders it after the accumulator's reads by every warp, which
  // lie before the barrier.
  auto issue = [&](int s, int buf, uint32_t nth) {
    tc::fence_after_sync();
    if (nth == (uint32_t)a.fault_stage) return;
    const uint64_t q = q_desc + (uint64_t)(s * kTile / 16), k = k_desc + (uint64_t)(buf * kTile / 16);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint64_t at = (uint64_t)(i / 4 * (128 * 128) / 16 + 2 * (i % 4));
      tc::mma_f8f6f4_ss(tmem + 128u * s, (kSum ? k : q) + at, (kSum ? q : k) + at, tc::kIdescQK, i > 0 ? 1u : 0u);
    }
    tc::commit(&sm.ready[s]);
  };
  // This thread's accumulator row and 64 of its columns.
  const uint32_t s_col = tmem + ((uint32_t)(warp & 3) << 21) + 64u * (warp >> 2);
  const int lane_row = 32 * (warp & 3) + lane, col0 = 64 * (warp >> 2);
  const float x_mul = a.inv_sqrt_d * kLog2e;
  const float e_bias = __uint_as_float(2u * D + smem_u32(sm.e));  // x 2^-149

  auto key_slot = [&](int t) { return t < k1 ? a.pages.slot(r, t) : -1LL; };
  auto load_key = [&](long long slot) { return load_half<D>(a.k + max(slot, 0LL) * W, half); };
  auto put_key = [&](const HalfRow<D>& h, long long slot, int buf) {
    expand_half<D>(h, k_tile + buf * kTile, row, half);
    uint32_t bits = __ballot_sync(0xffffffffu, slot >= 0) & 0x55555555u;  // a bit per pair of lanes
    bits = (bits | (bits >> 1)) & 0x33333333u;
    bits = (bits | (bits >> 2)) & 0x0F0F0F0Fu;
    bits = (bits | (bits >> 4)) & 0x00FF00FFu;
    bits = (bits | (bits >> 8)) & 0xFFFFu;
    if (lane == 0) sm.mask[buf][warp] = (uint16_t)bits;
  };
  auto flag_key = [&](long long slot, int t) {
    if (slot < 0 && t < k1 && half == 0) raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
  };

  uint32_t turn0 = 0, turn1 = 0;  // uses of each accumulator so far
  bool alive = true;              // no wait of this warp ran out; thread 0 issues while it is
  const int group0 = kSum ? 0 : in_row - chunk * c.groups, group1 = kSum ? c.groups : group0 + 1;
  for (int group = group0; group < group1; ++group) {
    const int q0 = group * kWinQueries;
    const int two = rows - q0 > 128 ? 2 : 1;  // accumulators in use
    // The first two key tiles on their way, then the group's queries: how far each sees,
    // 1 / l, and their bytes.
    long long slot = key_slot(k0 + row), next_slot = key_slot(k0 + kWinKeys + row);
    flag_key(slot, k0 + row);
    flag_key(next_slot, k0 + kWinKeys + row);
    HalfRow<D> h = load_key(slot);
    HalfRow<D> h2 = load_key(next_slot);
    HalfRow<D> hq[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int i = q0 + s * 128 + row;
      long long at = 0;
      const bool real = i < rows && query_of(a, r, i, n, &at) > 0;
      hq[s] = load_half<D>(a.q + (real ? at : 0) * W, half);
    }
    long long q_row = 0;
    const int end = q0 + tid < rows ? query_of(a, r, q0 + tid, n, &q_row) : 0;
    sm.end[tid] = end > 0 ? end : INT_MAX;
    if (tid == 0) sm.min_end = INT_MAX;
    put_key(h, slot, 0);
    put_key(h2, next_slot, 1);
    expand_half<D>(hq[0], q_tile, row, half);
    if (two == 2) expand_half<D>(hq[1], q_tile + kTile, row, half);
    next_slot = key_slot(k0 + 2 * kWinKeys + row);
    tc::fence_proxy_async_smem();
    __syncthreads();
    if (tid == 0 && alive) {
      issue(0, 0, turn0 + turn1);
      if (two == 2) issue(1, 0, turn0 + turn1 + 1);
    }
    const int least = __reduce_min_sync(0xffffffffu, end > 0 ? end : INT_MAX);
    if (lane == 0) atomicMin(&sm.min_end, least);
    if (kSum) {
      if (group == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
      float l = 0.f;
      const int used = (n + c.tiles * kWinKeys - 1) / (c.tiles * kWinKeys);
      const float* part = c.part + ((size_t)r * c.chunks * c.groups + group) * kWinQueries + tid;
      for (int j = 0; j < used; j += 8) {  // in order, 8 reads in flight
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = j + u < used ? __ldcg(part + (size_t)(j + u) * c.groups * kWinQueries) : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) l += x[u];
      }
      sm.inv[tid] = end > 0 && l > 0.f ? 1.f / l : 0.f;
    }
    __syncthreads();
    const int min_end = sm.min_end;
    float l[2] = {0.f, 0.f};

#pragma unroll 1
    for (int g = 0; g < tiles; ++g) {
      const int buf = g & 1, kb = k0 + g * kWinKeys;
      // Sign bits of tile g + 2 and the page of tile g + 3.
      slot = next_slot;
      const bool more = g + 2 < tiles;
      if (more) {
        flag_key(slot, kb + 2 * kWinKeys + row);
        h = load_key(slot);
        next_slot = key_slot(kb + 3 * kWinKeys + row);
      }
      const uint4 m = *reinterpret_cast<const uint4*>(sm.mask[buf]);
      const uint32_t mk[4] = {m.x, m.y, m.z, m.w};
      const bool whole = (mk[0] & mk[1] & mk[2] & mk[3]) == 0xffffffffu;
      const bool plain = kb + kWinKeys <= min_end && (kSum || whole);
      float sum = 0.f;
#pragma unroll 1
      for (int s = 0; s < two; ++s) {
        // A warp whose wait ran out reads no accumulator any more: what it holds need not be a
        // score, and would be no place of the table.
        alive = __all_sync(0xffffffffu, alive && mbar_wait(&sm.ready[s], (s ? turn1 : turn0) & 1, &sm.ctl, a.err));
        (s ? turn1 : turn0)++;
        tc::fence_after_sync();
        const uint32_t col = s_col + 128u * s;
        const float* inv = sm.inv + s * 128 + col0;
        float x = 0.f;
        if (!alive) {
        } else if (plain) {
          x = sum_columns<kSum, false>(col, e_bias, x_mul, inv, 0);
        } else {  // the columns this row pairs with: those that exist and are seen
          uint64_t on = 0;
          if (kSum) {
            const int t = kb + lane_row;
            for (int i = 0; i < 64; ++i) on |= (uint64_t)(t < sm.end[s * 128 + col0 + i]) << i;
          } else {
            const int lim = sm.end[s * 128 + lane_row] - (kb + col0);
            on = ((uint64_t)(col0 ? mk[3] : mk[1]) << 32 | (col0 ? mk[2] : mk[0])) &
                 (lim >= 64 ? ~0ull : lim <= 0 ? 0ull : (1ull << lim) - 1);
          }
          x = sum_columns<kSum, true>(col, e_bias, x_mul, inv, on);
        }
        if (kSum) {
          sum += x;
        } else if (s == 0) {
          l[0] += x;
        } else {
          l[1] += x;
        }
        if (kSum && s == two - 1 && col0) sm.half[buf][lane_row] = sum;
        tc::fence_before_sync();
        __syncthreads();
        if (tid == 0 && alive && g + 1 < tiles) issue(s, buf ^ 1, turn0 + turn1 + two - 1);
      }
      if (kSum && !col0) {
        float* out = sm.out + g * kWinKeys + lane_row;
        const float all = sum + sm.half[buf][lane_row];
        *out = group == 0 ? all : *out + all;
      }
      if (more) {  // both accumulators of tile g are complete: its buffer is free
        put_key(h, slot, buf);
        tc::fence_proxy_async_smem();
      }
    }
    if (!kSum) {
      __syncthreads();
      if (col0) sm.half[0][lane_row] = l[0], sm.half[1][lane_row] = l[1];
      __syncthreads();
      if (!col0) {
        float* part = c.part + (((size_t)r * c.chunks + chunk) * c.groups + group) * kWinQueries + lane_row;
        part[0] = l[0] + sm.half[0][lane_row];
        part[128] = l[1] + sm.half[1][lane_row];
      }
    }
    __syncthreads();
  }
  if (kSum) {
    const float* in = a.in + r * a.ld;
    float* out = a.out + r * a.ld;
    for (int t = k0 + tid; t < k1; t += kWinThreads) {
      // A key on a page outside the pool was scored as row 0 and gets nothing.
      const float w = a.pages.slot(r, t) >= 0 ? sm.out[t - k0] : 0.f;
      out[t] = fmaf(a.decay, in[t], w);
    }
  }
  if (tid == 0 && sm.ctl.flag) {  // let the products in flight land
    tc::commit(&sm.drain);
    mbar_drain(&sm.drain, 0, kWaitCycles);
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kWinTmemCols);
  }
}

template <int D>
constexpr int window_smem_bytes() {
  return (int)sizeof(WindowSmem<D>) + 1024;
}

template <int D>
inline cudaError_t window_setup_d() {
  cudaError_t e = cudaFuncSetAttribute(window_kernel<D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       window_smem_bytes<D>());
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(window_kernel<D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, window_smem_bytes<D>());
  return e;
}

// Once per device, before the first launch.
inline cudaError_t setup() {
  const cudaError_t e = window_setup_d<128>();
  return e == cudaSuccess ? window_setup_d<256>() : e;
}

constexpr int kSms = 148;  // of a B200; the plan, and so the scratch, does not depend on the device

// What a call launches and the scratch it needs.
struct Plan {
  bool few = false;   // the two streaming kernels
  int one = 0;        // or the first of them alone, a block a row of up to so many keys
  bool flat = false;  // else: the tensor-core window kernels, or those on the CUDA cores
  WindowArgs win = {};
  int unroll = 1, groups = 1;
  ChunkArgs c = {};
  size_t dist_bytes = 0, part_bytes = 0;  // at the front of the scratch, distances first
};

inline Plan plan(long long n_kv, long long rows, int head_dim, long long cap, bool flat) {
  Plan p;
  p.flat = flat;
  p.few = rows <= kMaxBatches * kBatch;
  if (!p.few && flat) {
    // Chunks of up to 16 tiles, shorter ones while the sums have fewer than 4 blocks an SM: two
    // rounds of the 2 that an SM holds at head_dim 128, four of the 1 at head_dim 256.
    p.win.groups = (int)((rows + kWinQueries - 1) / kWinQueries);
    p.win.tiles = kMaxChunkTiles;
    while (p.win.tiles > 2 && n_kv * ((cap + p.win.tiles * kWinKeys - 1) / (p.win.tiles * kWinKeys)) < 4 * kSms) p.win.tiles /= 2;
    p.win.chunks = (int)((cap + p.win.tiles * kWinKeys - 1) / (p.win.tiles * kWinKeys));
    p.part_bytes = (size_t)n_kv * p.win.chunks * p.win.groups * kWinQueries * sizeof(float);
    return p;
  }
  if (!p.few) {
    p.part_bytes = (size_t)(n_kv * rows) * sizeof(int2);
    return p;
  }
  p.c.batches = (int)((rows + kBatch - 1) / kBatch);
  // A row that one block holds is done by it, in one launch and without scratch: 8 rows of
  // 333 keys 4.4 us less a call from Python than in two (6.9 and 6.2 us on the device).
  // Blocks of 20 keys a thread would need 224 registers: 512 rows of 4100 keys 51 us against
  // 31 us in two.
  const int one = cap <= kThreads ? kThreads : cap <= 8 * kThreads ? 8 * kThreads : 0;
  if (one) {
    p.one = one;
    p.c.chunks = 1;
    return p;
  }
  const long long keys = n_kv * cap;
  // 8 keys a thread where that still gives every SM its blocks, else one.
  p.unroll = keys >= 2LL * kSms * kThreads * 8 ? 8 : 1;
  p.groups = p.unroll == 8 ? 2 : 1;
  const long long chunk = (long long)kThreads * p.unroll;
  p.c.chunks = (int)((cap + chunk - 1) / chunk);
  const long long whole = (cap + 8 * kThreads - 1) / (8 * kThreads) * (8 * kThreads);
  p.c.dist_ld = (int)whole;
  p.dist_bytes = (size_t)n_kv * p.c.batches * whole * (head_dim == 256 ? 8 : 4);
  p.part_bytes = (size_t)n_kv * p.c.chunks * p.c.batches * kBatch * sizeof(int2);
  return p;
}

template <int D, bool kFlat>
inline cudaError_t launch_few(const Args& a, Plan p, uint8_t* scratch, cudaStream_t st) {
  const long long cap = (long long)a.pages.num_blocks * a.pages.block_size;
  p.c.dist = scratch;
  p.c.part = reinterpret_cast<int2*>(scratch + p.dist_bytes);
  const unsigned grid = (unsigned)((long long)a.n_kv * p.c.chunks);
  constexpr int U = D == 128 ? 4 : 2;
  if (p.one) {
    if (p.one == kThreads) {
      score_kernel<D, kFlat, 1, 1, true><<<grid, kThreads, 0, st>>>(a, p.c);
    } else {
      score_kernel<D, kFlat, U, 8 / U, true><<<grid, kThreads, 0, st>>>(a, p.c);
    }
    return cudaGetLastError();
  }
  if (p.unroll == 8) {
    score_kernel<D, kFlat, U, 8 / U, false><<<grid, kThreads, 0, st>>>(a, p.c);
  } else {
    score_kernel<D, kFlat, 1, 1, false><<<grid, kThreads, 0, st>>>(a, p.c);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const long long block = 4LL * kThreads * p.groups;
  const int per_row = (int)((cap + block - 1) / block);
  const bool vec = a.ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.in) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)a.n_kv * per_row));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = p.groups == 2 ? sum_kernel<D, kFlat, 2> : sum_kernel<D, kFlat, 1>;
  e = cudaLaunchKernelEx(&cfg, kernel, a, p.c, kThreads * p.unroll, per_row, vec);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

template <int D>
inline cudaError_t launch_window(const Args& a, Plan p, uint8_t* scratch, cudaStream_t st) {
  p.win.part = reinterpret_cast<float*>(scratch);
  const long long blocks = (long long)a.n_kv * p.win.chunks;
  window_kernel<D, false><<<(unsigned)(blocks * p.win.groups), kWinThreads, window_smem_bytes<D>(), st>>>(a, p.win);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kWinThreads);
  cfg.dynamicSmemBytes = window_smem_bytes<D>();
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, window_kernel<D, true>, a, p.win);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

// Whether no exponential of the call can reach the clamp.
inline bool is_flat(float inv_sqrt_d, int head_dim) { return 2.f * std::fabs(inv_sqrt_d) * head_dim <= -kExpClamp; }

template <int D>
inline cudaError_t launch_d(Args a, uint8_t* scratch, cudaStream_t st) {
  const long long rows = (long long)a.kv_group * a.n_q;
  const long long cap = (long long)a.pages.num_blocks * a.pages.block_size;
  const Plan p = plan(a.n_kv, rows, D, cap, is_flat(a.inv_sqrt_d, D));
  if (p.few) return p.flat ? launch_few<D, true>(a, p, scratch, st) : launch_few<D, false>(a, p, scratch, st);
  if (p.flat) return launch_window<D>(a, p, scratch, st);
  a.stats = reinterpret_cast<int2*>(scratch);
  const int per_row = (int)((cap + kThreads - 1) / kThreads);
  window_stats_kernel<D><<<(unsigned)(a.n_kv * rows), kThreads, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  window_sum_kernel<D><<<(unsigned)(a.n_kv * (long long)per_row), kThreads, 0, st>>>(a, per_row);
  return cudaGetLastError();
}

inline cudaError_t launch(const Args& a, int head_dim, uint8_t* scratch, cudaStream_t st) {
  return head_dim == 256 ? launch_d<256>(a, scratch, st) : launch_d<128>(a, scratch, st);
}

}  // namespace kweights
}  // namespace hyp
