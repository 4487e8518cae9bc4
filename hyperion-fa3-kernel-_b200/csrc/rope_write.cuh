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

#include <algorithm>

#include "cache_pages.cuh"
#include "kv_write.cuh"

namespace hyp {
namespace rope {

constexpr int kWarpsPerBlock = 8;
// Query rows of one lane group in flight at once: 64 bytes a thread and 4 blocks an SM.
// (32768 tokens of 32 + 8 heads of 128, bf16: 98 us; 4 rows and 3 blocks 102 us, 4 rows and
// 2 blocks 118 us, 1 row and 5 blocks 146 us: the issue slots are as busy as HBM.  At the 64
// registers of 4 blocks every instance spills, 84 to 116 bytes of stores a thread.)
template <typename T>
constexpr int kUnroll = sizeof(T) == 2 ? 2 : 1;
constexpr int kBlocksPerSm = 4;

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
  Pages pages;
  long long bt_rows;
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

// Cache rows and query heads are int32 to the forward; beyond, the products with rows or pages
// a head could wrap.
constexpr long long kMaxHeads = 0x7fffffff;

// Query row of (sequence b, head h) for token `tok` at `pos`, or -1.
__device__ __forceinline__ long long q_row_of(const Args& a, int tok, int b, int pos, int h) {
  const int qi = a.q_idx ? __ldg(a.q_idx + tok) : (a.seq_q == 1 ? 0 : pos);
  const long long head = (long long)b * a.n_heads + h;
  if (head > kMaxHeads || qi < 0 || qi >= a.seq_q) return -1;
  const long long row = head * a.seq_q + qi;
  return row < a.q_rows ? row : -1;
}

// Pool row of cache row kv for token `tok` at `pos`, or -1 with the error raised by `flag`.
__device__ __forceinline__ long long kv_row_of(const Args& a, int tok, int pos, int h, long long kv, bool flag, int* slot) {
  const int t = a.slots ? __ldg(a.slots + (a.slots_per_head ? (long long)tok * a.n_kv_heads + h : (long long)tok)) : pos;
  *slot = t;
  if (t < 0 || t >= a.pages.capacity() || kv > kMaxHeads || (a.pages.tables && kv >= a.bt_rows) ||
      (a.slot_positions && kv >= a.slot_rows)) {
    if (flag) raise_error(a.err, HYPERION_DEVERR_BAD_ITEM);
    return -1;
  }
  const long long row = a.pages.slot(kv, t);
  if (row < 0 && flag) raise_error(a.err, HYPERION_DEVERR_BAD_BLOCK);
  return row;
}

__device__ __forceinline__ float v_scale_of(const Args& a, long long kv, long long row) {
  const long long si = a.v_scale_numel == 1 ? 0 : (a.v_scale_numel == a.pool_rows ? row : kv % a.v_scale_numel);
  return __ldg(a.v_scale + si);
}

__device__ __forceinline__ uint32_t v_code(float v, float scale) {
  float y = __fdiv_rn(v, scale);
  if (y == y) y = fminf(fmaxf(y, -448.f), 448.f);
  return kvw::e4m3_code(y);
}

// ---------------------------------------------------------------------------
// The vector kernel: rotary_dim a multiple of 16, inputs on 16-byte boundaries.
//
// D / 16 lanes share a row, so a warp holds 4 rows of 128 dims or 2 of 256.  Lane j of a
// row takes 16 dims as two runs of 8, each one 16-byte load of 16-bit values and one byte
// of signs: the run of pair members a and that of members b (half layout), or 16
// neighbouring dims (interleaved).  Either way its pairs are 8j .. 8j + 7, and the warp
// keeps one token's cos / sin in registers for all the heads it takes.
// ---------------------------------------------------------------------------
template <typename T>
struct Run8 {
  uint4 x[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Run8<T> load8(const T* p) {
  Run8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.x[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return r;
}

// Eight values as pairs, for the packed f32x2 instructions (half the instructions of the
// kernel's products and sums, which its issue slots would otherwise bound).
struct Pairs8 {
  float2 p[4];
  __device__ __forceinline__ float at(int i) const { return i & 1 ? p[i / 2].y : p[i / 2].x; }
};

template <typename T>
__device__ __forceinline__ Pairs8 widen8(const Run8<T>& r) {
  const T* x = reinterpret_cast<const T*>(r.x);
  Pairs8 f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f.p[i] = make_float2(kvw::to_f32<T>(x[2 * i]), kvw::to_f32<T>(x[2 * i + 1]));
  return f;
}

// Signs of x*c + y*s (x*c - y*s where kMinus) for 8 elements as a byte (element 0 in bit 0, 1
// where >= 0).  The sign bits of the rounded sums are shifted in one by one; a sum that is
// zero or NaN sends the run to the exact form.
template <bool kMinus>
__device__ __forceinline__ uint32_t sign_byte(const Pairs8& x, const Pairs8& c, const Pairs8& y, const Pairs8& s) {
  uint32_t neg = 0;
  bool clear = true;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    const float2 u = __fmul2_rn(x.p[i], c.p[i]), w = __fmul2_rn(y.p[i], s.p[i]);
    const float2 d = kMinus ? __ffma2_rn(w, make_float2(-1.f, -1.f), u) : __fadd2_rn(u, w);
    neg = __funnelshift_l(__float_as_uint(d.y), neg, 1);
    neg = __funnelshift_l(__float_as_uint(d.x), neg, 1);
    clear = clear && fabsf(d.x) > 0.f && fabsf(d.y) > 0.f;
  }
  uint32_t up = ~neg & 0xFFu;
  if (!clear) {
    up = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) up |= (sum_is_nonneg(x.at(i), c.at(i), y.at(i), kMinus ? -s.at(i) : s.at(i)) ? 1u : 0u) << i;
  }
  return up;
}

__device__ __forceinline__ uint32_t plain_byte(const Pairs8& x) {
  uint32_t up = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) up |= (x.at(i) >= 0.f ? 1u : 0u) << i;
  return up;
}

// Both sign bytes of a lane's 16 dims.
template <typename T, bool kHalf>
__device__ __forceinline__ void turn16(const Run8<T>& r0, const Run8<T>& r1, const Pairs8& c, const Pairs8& s, bool turned,
                                       uint32_t& b0, uint32_t& b1) {
  const Pairs8 x = widen8<T>(r0), y = widen8<T>(r1);
  if (!turned) {
    b0 = plain_byte(x);
    b1 = plain_byte(y);
  } else if (kHalf) {
    b0 = sign_byte<true>(x, c, y, s);
    b1 = sign_byte<false>(y, c, x, s);
  } else {
    // neighbours: members a in the even places, b in the odd ones
    Pairs8 p, q;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      p.p[i] = make_float2(x.p[2 * i].x, x.p[2 * i + 1].x);
      q.p[i] = make_float2(x.p[2 * i].y, x.p[2 * i + 1].y);
      p.p[i + 2] = make_float2(y.p[2 * i].x, y.p[2 * i + 1].x);
      q.p[i + 2] = make_float2(y.p[2 * i].y, y.p[2 * i + 1].y);
    }
    uint32_t u = sign_byte<true>(p, c, q, s), w = sign_byte<false>(q, c, p, s);
    // bit i of u to bit 2i, of w to bit 2i + 1
    u = (u | (u << 4)) & 0x0F0Fu;
    u = (u | (u << 2)) & 0x3333u;
    u = (u | (u << 1)) & 0x5555u;
    w = (w | (w << 4)) & 0x0F0Fu;
    w = (w | (w << 2)) & 0x3333u;
    w = (w | (w << 1)) & 0x5555u;
    const uint32_t both = u | (w << 1);
    b0 = both & 0xFFu;
    b1 = both >> 8;
  }
}

// e4m3 codes of RN(v / scale), saturated, for 8 values, four a word.  v times the rounded
// reciprocal is within 1.5 steps of the quotient, so it has the quotient's code unless a
// border between two codes lies that near: borders have at most 5 significant bits, so the
// low 19 bits of such a number are within 2 of 0.  Those runs, and scales whose reciprocal
// is not an ordinary number, are divided; a scale that is a power of two never is, there
// the product is the quotient.
__device__ __forceinline__ void v_codes8(const Pairs8& v, float scale, float recip, uint32_t (&w)[2]) {
  float q[8];
  const bool ordinary = fabsf(scale) >= 0x1p-60f && fabsf(scale) <= 0x1p60f;
  const bool power = (__float_as_uint(scale) & 0x7FFFFFu) == 0;
  bool near = false;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 x = __fmul2_rn(v.p[i / 2], make_float2(recip, recip));
    q[i] = x.x, q[i + 1] = x.y;
    near = near || ((__float_as_uint(x.x) + 2) & 0x7FFFFu) <= 4 || ((__float_as_uint(x.y) + 2) & 0x7FFFFu) <= 4;
  }
  if (!ordinary || (near && !power)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(v.at(i), scale);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint16_t lo, hi;  // the second source lands in the low byte; saturation is the clamp to +-448
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(q[4 * i + 1]), "f"(q[4 * i]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(q[4 * i + 3]), "f"(q[4 * i + 2]));
    w[i] = (uint32_t)lo | (uint32_t)hi << 16;
  }
}

// Warp `wid` takes token wid / parts and the row units [part * per, (part + 1) * per) of
// its n_heads query heads and n_kv_heads (K, V) pairs.
template <int D, typename T, bool kHalf>
__global__ void __launch_bounds__(32 * kWarpsPerBlock, kBlocksPerSm) rope_write_vec_kernel(Args a, int parts, int per) {
  constexpr int W = D / 32;
  constexpr int G = D / 16;  // lanes a row
  constexpr int R = 32 / G;  // rows a warp
  constexpr int U = kUnroll<T>;
  __shared__ __align__(16) uint8_t s_bytes[kWarpsPerBlock][U * R][D / 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = lane % G, g = lane / G;
  const long long wid = (long long)blockIdx.x * kWarpsPerBlock + warp;
  const int tok = (int)(wid / parts);
  const int part = (int)(wid - (long long)tok * parts);
  if (tok >= a.n_tokens) return;
  const int b = __ldg(a.seq_ids + tok);
  const int pos = __ldg(a.positions + tok);
  if (b < 0 || pos < 0 || (a.rot > 0 && pos >= a.n_positions)) {
    if (lane == 0) raise_error(a.err, HYPERION_DEVERR_BAD_ITEM);
    return;
  }
  // Runs of this lane in a row, in units of 8 dims.
  const int turning = a.rot / 16;  // lanes whose dims turn
  const bool turned = j < turning;
  int c0 = 2 * j, c1 = 2 * j + 1;
  if (kHalf && turned) {
    c0 = j;
    c1 = turning + j;
  }
  Pairs8 c, s;
  if (turned) {
    const float4* cs = reinterpret_cast<const float4*>(a.table + (long long)pos * a.rot) + 2 * j;
    const float4* sn = reinterpret_cast<const float4*>(a.table + (long long)pos * a.rot + a.rot / 2) + 2 * j;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 p = __ldg(cs + i), q = __ldg(sn + i);
      c.p[2 * i] = make_float2(p.x, p.y), c.p[2 * i + 1] = make_float2(p.z, p.w);
      s.p[2 * i] = make_float2(q.x, q.y), s.p[2 * i + 1] = make_float2(q.z, q.w);
    }
  }
  uint8_t(*buf)[D / 8] = s_bytes[warp];

  const int u0 = part * per, u1 = min(u0 + per, a.n_heads + a.n_kv_heads);
  const int q1 = min(u1, a.n_heads);
  const T* q = static_cast<const T*>(a.q) + tok * a.q_ts;
  for (int base = u0; base < q1; base += U * R) {
    Run8<T> r[U][2];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = min(base + i * R + g, q1 - 1);  // rows beyond the last are not stored
      r[i][0] = load8<T>(q + h * a.q_hs + 8 * c0);
      r[i][1] = load8<T>(q + h * a.q_hs + 8 * c1);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      uint32_t b0, b1;
      turn16<T, kHalf>(r[i][0], r[i][1], c, s, turned, b0, b1);
      buf[i * R + g][c0] = (uint8_t)b0;
      buf[i * R + g][c1] = (uint8_t)b1;
    }
    __syncwarp();
    // The U * R rows in pieces of 16 bytes.
    constexpr int kPieces = U * R * (D / 128);
    if (lane < kPieces) {
      const int row = lane / (D / 128), piece = lane % (D / 128);
      const int h = base + row;
      if (h < q1) {
        const long long out = q_row_of(a, tok, b, pos, h);
        if (out < 0) {
          raise_error(a.err, HYPERION_DEVERR_BAD_ITEM);
        } else {
          *reinterpret_cast<uint4*>(a.q_words + out * W + 4 * piece) = *reinterpret_cast<const uint4*>(&buf[row][16 * piece]);
        }
      }
    }
    __syncwarp();
  }

  for (int base = max(u0, a.n_heads); base < u1; base += R) {
    const int h = min(base + g, u1 - 1) - a.n_heads;
    const T* kr = static_cast<const T*>(a.k) + tok * a.k_ts + h * a.k_hs;
    const T* vr = static_cast<const T*>(a.v) + tok * a.v_ts + h * a.v_hs + 16 * j;
    const Run8<T> k0 = load8<T>(kr + 8 * c0), k1 = load8<T>(kr + 8 * c1);
    const Run8<T> v0 = load8<T>(vr), v1 = load8<T>(vr + 8);
    const long long kv = (long long)b * a.n_kv_heads + h;
    int slot = 0;
    const long long out = base + g < u1 ? kv_row_of(a, tok, pos, h, kv, j == 0, &slot) : -1;
    uint32_t b0, b1;
    turn16<T, kHalf>(k0, k1, c, s, turned, b0, b1);
    buf[g][c0] = (uint8_t)b0;
    buf[g][c1] = (uint8_t)b1;
    __syncwarp();
    if (out >= 0) {
      if (j < D / 128)
        *reinterpret_cast<uint4*>(a.k_cache + out * W + 4 * j) = *reinterpret_cast<const uint4*>(&buf[g][16 * j]);
      if (j == 0 && a.slot_positions) a.slot_positions[kv * a.pages.capacity() + slot] = pos;
      const float scale = v_scale_of(a, kv, out);
      const float recip = __frcp_rn(scale);
      uint32_t lo[2], hi[2];
      v_codes8(widen8<T>(v0), scale, recip, lo);
      v_codes8(widen8<T>(v1), scale, recip, hi);
      *reinterpret_cast<uint4*>(a.v_cache + out * D + 16 * j) = make_uint4(lo[0], lo[1], hi[0], hi[1]);
    }
    __syncwarp();
  }
}

// ---------------------------------------------------------------------------
// The scalar kernel: any even rotary_dim, any alignment and stride.  One warp per (token,
// query head) and per (token, KV head); lane l takes dims l, l + 32, ..., so a ballot is
// one sign word.  (32768 tokens of 32 + 8 heads of 128, bf16: 625 us, the vector kernel 98.)
// ---------------------------------------------------------------------------
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
  const long long kv = (long long)b * a.n_kv_heads + h;
  long long out_row;
  if (is_q) {
    out_row = q_row_of(a, tok, b, pos, h);
    if (out_row < 0) {
      if (lane == 0) raise_error(a.err, HYPERION_DEVERR_BAD_ITEM);
      return;
    }
  } else {
    int slot;
    out_row = kv_row_of(a, tok, pos, h, kv, lane == 0, &slot);
    if (out_row < 0) return;
    if (a.slot_positions && lane == 0) a.slot_positions[kv * a.pages.capacity() + slot] = pos;
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
  const float scale = v_scale_of(a, kv, out_row);
  const T* vr = static_cast<const T*>(a.v) + tok * a.v_ts + h * a.v_hs;
#pragma unroll
  for (int w = 0; w < W; ++w)
    a.v_cache[out_row * D + 32 * w + lane] = (uint8_t)v_code(kvw::to_f32<T>(vr[32 * w + lane]), scale);
}

inline bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int D, typename T>
inline cudaError_t launch_t(const Args& a, int n_sm, cudaStream_t st) {
  constexpr long long kPer16 = 16 / sizeof(T);
  const long long units = a.n_heads + a.n_kv_heads;
  const bool vec = a.rot % 16 == 0 && on16(a.table) && on16(a.q) && on16(a.k) && on16(a.v) &&
                   (a.q_ts | a.q_hs | a.k_ts | a.k_hs | a.v_ts | a.v_hs) % kPer16 == 0;
  if (vec) {
    // Enough warps to fill the device, no more than one round of rows each.
    constexpr int R = 512 / D;
    const long long want = (32LL * n_sm + a.n_tokens - 1) / a.n_tokens;
    const long long parts0 = std::max(1LL, std::min(want, (units + R - 1) / R));
    const int per = (int)((((units + parts0 - 1) / parts0) + R - 1) / R * R);
    const int parts = (int)((units + per - 1) / per);
    const unsigned grid = (unsigned)(((long long)a.n_tokens * parts + kWarpsPerBlock - 1) / kWarpsPerBlock);
    if (a.interleaved) {
      rope_write_vec_kernel<D, T, false><<<grid, 32 * kWarpsPerBlock, 0, st>>>(a, parts, per);
    } else {
      rope_write_vec_kernel<D, T, true><<<grid, 32 * kWarpsPerBlock, 0, st>>>(a, parts, per);
    }
  } else {
    const unsigned grid = (unsigned)((a.n_tokens * units + kWarpsPerBlock - 1) / kWarpsPerBlock);
    rope_write_kernel<D, T><<<grid, 32 * kWarpsPerBlock, 0, st>>>(a);
  }
  return cudaGetLastError();
}

template <int D>
inline cudaError_t launch_d(const Args& a, int in_dtype, int n_sm, cudaStream_t st) {
  if (in_dtype == HYPERION_DTYPE_F32) return launch_t<D, float>(a, n_sm, st);
  if (in_dtype == HYPERION_DTYPE_BF16) return launch_t<D, __nv_bfloat16>(a, n_sm, st);
  return launch_t<D, __half>(a, n_sm, st);
}

inline cudaError_t launch(const Args& a, int head_dim, int in_dtype, int n_sm, cudaStream_t st) {
  return head_dim == 256 ? launch_d<256>(a, in_dtype, n_sm, st) : launch_d<128>(a, in_dtype, n_sm, st);
}

}  // namespace rope
}  // namespace hyp
