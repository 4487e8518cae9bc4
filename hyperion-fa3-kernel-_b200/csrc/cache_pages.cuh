// cache_pages.cuh -- where the cache operators find slot t of cache row r.
#pragma once

#include <algorithm>

#include "common.cuh"

namespace hyp {

// t / d for 0 <= t < 2^31 by one multiplication (a 32-bit division by a runtime value is
// about 20 instructions): with 2^s >= d and m = ceil(2^(31+s) / d) < 2^32, floor(t m /
// 2^(31+s)) is exact because the error t (m d - 2^(31+s)) / (d 2^(31+s)) is below t / 2^(31+s)
// <= t / (2^31 d) < 1 / d.
struct FastDiv {
  uint32_t d = 1, mul = 0, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t n) : d(n) {
    while ((1ULL << shift) < n) ++shift;
    mul = n == 1 ? 0 : (uint32_t)(((1ULL << (31 + shift)) + n - 1) / n);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t t) const {
    return d == 1 ? t : __umulhi(2 * t, mul) >> shift;
  }
};

struct Pages {
  const int32_t* tables = nullptr;  // [rows, num_blocks], or nullptr: page p of row r is r * num_blocks + p
  uint32_t pool_blocks = 0;  // of the pool, at most 2^31: page ids are int32
  int block_size = 1, num_blocks = 1;
  FastDiv div;

  Pages() = default;
  Pages(const int32_t* tables_, long long tables_numel, int block_size_, int num_blocks_, long long pool_rows)
      : tables(tables_numel > 0 ? tables_ : nullptr),
        pool_blocks((uint32_t)std::min<long long>(pool_rows / block_size_, 1LL << 31)),
        block_size(block_size_),
        num_blocks(num_blocks_),
        div((uint32_t)block_size_) {}

  __device__ __forceinline__ int capacity() const { return block_size * num_blocks; }  // int32: checked on the host

  // Pool row of slot t (< capacity) of row r, or -1 when its page lies outside the pool.
  __device__ __forceinline__ long long slot(long long r, int t) const {
    const int page = (int)div.quotient((uint32_t)t);
    const int off = t - page * block_size;
    const long long at = r * num_blocks + page;
    if (tables) {
      const uint32_t id = (uint32_t)__ldg(tables + at);
      return id < pool_blocks ? (long long)id * block_size + off : -1;
    }
    return at < (long long)pool_blocks ? at * block_size + off : -1;
  }

  // A row's context length, clamped to [0, capacity]; `flag` raises the length's errors.
  __device__ __forceinline__ int context(int ctx, uint32_t* err, bool flag) const {
    if (ctx < 0) {
      if (flag) raise_error(err, HYPERION_DEVERR_NEG_CTX);
      return 0;
    }
    if (ctx > capacity()) {
      if (flag) raise_error(err, HYPERION_DEVERR_CTX_OVERFLOW);
      return capacity();
    }
    return ctx;
  }
};

}  // namespace hyp
