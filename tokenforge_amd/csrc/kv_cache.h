// The paged key-value cache as its kernels address it, and the checks their C entries share.
#pragma once

#include "fp8_rows.h"

namespace tf {

// Exact division of n < 2^31 by a page size: n / d = (n * mul) >> (31 + shift), mul = ceil(2^(31 + shift) / d)
// with 2^(shift - 1) < d <= 2^shift. mul d exceeds 2^(31 + shift) by less than d <= 2^shift, so the quotient's
// excess n (mul d - 2^(31 + shift)) / (d 2^(31 + shift)) stays below 1 / d for n < 2^31, and mul <= 2^32 - 1
// (d = 1: mul = 2^31).
struct PageDiv {
  uint32_t mul;
  uint32_t shift;
  uint32_t page;
};

inline PageDiv page_div(uint32_t d) {
  uint32_t shift = 0;
  while ((uint64_t(1) << shift) < d) ++shift;
  return PageDiv{(uint32_t)(((uint64_t(1) << (31 + shift)) + d - 1) / d), shift, d};
}

__host__ __device__ __forceinline__ uint32_t div_page(uint32_t n, const PageDiv& p) {
  return (uint32_t)(((uint64_t)n * p.mul) >> (31 + p.shift));
}

// "" or what is wrong with a cache, as the caller's message.
std::string kv_cache_error(const tf_kv_cache* c, int32_t dtype);

constexpr int64_t kMaxTokenStride = int64_t(1) << 24;  // elements: 16 tokens' byte offsets stay in 31 bits

}  // namespace tf
