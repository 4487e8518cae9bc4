// rope_write.cuh -- rotary positions on new queries and keys, fused with the packing of
// both and with the cache write: the step between a layer's projections and the forward.
//
// For the pair (a, b) of a head's rotated dims and the table's cos / sin of the token's
// position,
//   r_a = x_a cos - x_b sin,   r_b = x_b cos + x_a sin,
// and only the signs of r_a and r_b are kept (bit = 1 where r >= 0).  The sign is that
// of the exact sum of the two products (f32 table values, inputs of f32 or less), so it
// does not depend on how a sum next to zero is rounded: see sum_is_nonneg.  V becomes
// e4m3 codes as in kv_write.cuh.
#pragma once

#include "kv_write.cuh"

namespace hyp {
namespace rope {

constexpr int kWarpsPerBlock = 8;

struct Args {
  const void* q;  // [n_tokens, n_heads, D], strides in elements
  const void* k;  // [n_tokens, n_kv_heads, D]
  const void* v;
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  int n_tokens, n_heads, n_kv_heads;
  const int32_t* seq_ids;
  const int32_t* positions;
  const int32_t* q_idx;  // nullptr: 0 when seq_q is 1, else the position
  const int32_t* slots;  // nullptr: the position; [n_tokens] or [n_tokens, n_kv_heads]
  int slots_per_head;
  const float* table;  // [n_positions, 2, rot / 2]: cos row, sin row
  int n_positions, rot, interleaved;
  const int32_t* block_tables;
  long long bt_rows;
  int block_size, num_blocks;
  const float* v_scale;
  long long v_scale_numel;
  uint32_t* q_words;
  long long q_rows;
  int seq_q;
  uint32_t* k_cache;
  uint8_t* v_cache;
  long long pool_rows;
  int32_t* slot_positions;  // nullptr or [slot_rows, num_blocks * block_size]
  long long slot_rows;
  uint32_t* err;
};

// x*c + y*s >= 0 for the exact sum.  Rounding is monotone, so the rounded products
// compare as the exact ones unless they are equal; then (and for NaN) the products are
// taken in f64, where they are exact, and their sum has the exact sum's sign.
__device__ __forceinline__ bool sum_is_nonneg(float x, float c, float y, float s) {
  const float d = __fadd_rn(__fmul_rn(x, c), __fmul_rn(y, s));
  if (d > 0.f) return true;
  if (d < 0.f) return false;
  return __dadd_rn(__dmul_rn((double)x, (double)c), __dmul_rn((double)y, (double)s)) >= 0.0;
}

// One warp per (token, head) of Q and per (token, KV head) of K and V.  Lane l takes
// dims l, l + 32, ..., so a ballot is one sign word.
template <int D, typename T>
__global__ void __launch_bounds__(32 * kWarpsPerBlock) rope_write_kernel(Args a) {
  constexpr int W = D / 32;
  const int lane = threadIdx.x & 31;
  const int heads = a.n_heads + a.n_kv_heads;
  const long long wid = (long long)blockIdx.x * kWarpsPerBlock + (threadIdx.x >> 5);
  if (wid >= (long long)a.n_tokens * heads) return;
  const int tok = (int)(wid / heads);
  const int hh = (int)(wid - (long long)tok * heads);
  const int b = __ldg(a.seq_ids + tok);
  const int pos = __ldg(a.positions + tok);
  if (b < 0 || pos < 0 || (a.rot > 0 && pos >= a.n_positions)) {
    if (lane == 0) raise_error(a.err, HYPERION_DEVERR_BAD_ITEM);
    return;
  }
  const bool is_q = hh < a.n_heads;
  const int h = is_q ? hh : hh - a.n_heads;
  const T* row = is_q ? static_cast<const T*>(a.q) + tok * a.q_ts + h * a.q_hs
                      : static_cast<const T*>(a.k) + tok * a.k_ts + h * a.k_hs;
  long long out_row, kv = 0;
  if (is_q) {
    const int qi = a.q_idx ? __ldg(a.q_idx + tok) : (a.seq_q == 1 ? 0 : pos);
    out_row = ((long long)b * a.n_heads + h) * a.seq_q + qi;
    if (qi < 0 || qi >= a.seq_q || out_row >= a.q_rows) {
      if (lane == 0) raise_error(a.err, HYPERION_DEVERR_BAD_ITEM);
      return;
    }
  } else {
    kv = (long long)b * a.n_kv_heads + h;
    const int t = a.slots ? __ldg(a.slots + (a.slots_per_head ? (long long)tok * a.n_kv_heads + h : (long long)tok)) : pos;
    const long long cap = (long long)a.num_blocks * a.block_size;
    if (t < 0 || (long long)t >= cap || (a.block_tables && kv >= a.bt_rows) ||
        (a.slot_positions && kv >= a.slot_rows)) {
      if (lane == 0) raise_error(a.err, HYPERION_DEVERR_BAD_ITEM);
      return;
    }
    const int page = t / a.block_size;
    const long long id =
        a.block_tables ? (long long)__ldg(a.block_tables + kv * a.num_blocks + page) : kv * a.num_blocks + page;
    if (id < 0 || id >= a.pool_rows / a.block_size) {
      if (lane == 0) raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
      return;
    }
    out_row = id * a.block_size + (t - page * a.block_size);
    if (a.slot_positions && lane == 0) a.slot_positions[kv * cap + t] = pos;
  }
  const int half = a.rot / 2;
  const float* cs = a.table + (long long)pos * a.rot;
  uint32_t word = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int d = 32 * w + lane;
    const float x = kvw::to_f32<T>(row[d]);
    bool up;
    if (d >= a.rot) {
      up = x >= 0.f;
    } else {
      const int pair = a.interleaved ? d >> 1 : (d < half ? d : d - half);
      const bool second = a.interleaved ? (d & 1) : d >= half;
      const int other = a.interleaved ? (d ^ 1) : (second ? d - half : d + half);
      const float y = kvw::to_f32<T>(row[other]);
      const float s = __ldg(cs + half + pair);
      up = sum_is_nonneg(x, __ldg(cs + pair), y, second ? s : -s);
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, up);
    if (lane == w) word = bits;
  }
  if (lane < W) (is_q ? a.q_words : a.k_cache)[out_row * W + lane] = word;
  if (is_q) return;
  const long long si = a.v_scale_numel == 1 ? 0 : (a.v_scale_numel == a.pool_rows ? out_row : kv % a.v_scale_numel);
  const float scale = __ldg(a.v_scale + si);
  const T* vr = static_cast<const T*>(a.v) + tok * a.v_ts + h * a.v_hs;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    float y = __fdiv_rn(kvw::to_f32<T>(vr[32 * w + lane]), scale);
    if (y == y) y = fminf(fmaxf(y, -448.f), 448.f);
    a.v_cache[out_row * D + 32 * w + lane] = (uint8_t)kvw::e4m3_code(y);
  }
}

template <int D>
inline cudaError_t launch_d(const Args& a, int in_dtype, cudaStream_t st) {
  const long long warps = (long long)a.n_tokens * (a.n_heads + a.n_kv_heads);
  const unsigned grid = (unsigned)((warps + kWarpsPerBlock - 1) / kWarpsPerBlock);
  if (in_dtype == HYPERION_DTYPE_F32) {
    rope_write_kernel<D, float><<<grid, 32 * kWarpsPerBlock, 0, st>>>(a);
  } else if (in_dtype == HYPERION_DTYPE_BF16) {
    rope_write_kernel<D, __nv_bfloat16><<<grid, 32 * kWarpsPerBlock, 0, st>>>(a);
  } else {
    rope_write_kernel<D, __half><<<grid, 32 * kWarpsPerBlock, 0, st>>>(a);
  }
  return cudaGetLastError();
}

inline cudaError_t launch(const Args& a, int head_dim, int in_dtype, cudaStream_t st) {
  return head_dim == 256 ? launch_d<256>(a, in_dtype, st) : launch_d<128>(a, in_dtype, st);
}

}  // namespace rope
}  // namespace hyp
