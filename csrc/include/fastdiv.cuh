// Division by a number that the host knows.
#pragma once
#include <cstdint>

namespace meshy {

// n / d for n < 2^31, as (n m) >> s with m = ceil(2^s / d), s = 31 + ceil(log2 d) (Granlund and Montgomery, 1994).
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t d_) : d(d_), s(31) {
    while ((1ull << (s - 31)) < d) ++s;
    m = (uint32_t)(((1ull << s) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> s); }
};

}  // namespace meshy
