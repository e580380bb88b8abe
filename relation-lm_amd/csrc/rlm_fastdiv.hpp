// Division of 32-bit unsigned numbers by a number fixed at launch.
#pragma once

#include <cstdint>

namespace rlm {

// n / d for every n < 2^31 and 1 <= d < 2^31, as one high multiplication and a shift: with
// s = ceil(log2 d) and m = floor(2^(31+s) / d) + 1 (below 2^32), the product m n exceeds
// n 2^(31+s) / d by less than 2^(31+s) / d, so no quotient is passed.  d = 1: m = 2^31 + 1.
struct FastDiv {
  uint32_t d = 1, mul = 0, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t divisor) : d(divisor) {
    uint32_t s = 0;
    while ((uint64_t(1) << s) < d) ++s;
    mul = static_cast<uint32_t>((uint64_t(1) << (31 + s)) / d + 1);
    shift = s;
  }
  __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> 31 >> shift);
  }
  __host__ __device__ __forceinline__ uint32_t div(uint32_t n, uint32_t& rest) const {
    const uint32_t q = div(n);
    rest = n - q * d;
    return q;
  }
};

}  // namespace rlm
