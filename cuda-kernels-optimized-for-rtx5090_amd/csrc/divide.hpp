// Division by numbers that the host knows.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rw {

// Of n with 0 <= n < 2^31: with 2^(s - 1) < d <= 2^s, n * (floor(2^(31 + s) / d) + 1) is more than n * 2^(31 + s) / d by
// at most n <= 2^31, less than the 2^(31 + s) / d that a quotient's last fraction leaves. (An integer division is some
// 30 instructions, and a workgroup's first load waited for ten of them.)
struct Divisor {
  uint32_t d, inverse;
  int shift;
  __device__ __forceinline__ unsigned of(unsigned n) const {
    return (unsigned)(((uint64_t)(2u * n) * inverse) >> 32) >> shift;
  }
  // n becomes its quotient; the remainder is returned
  __device__ __forceinline__ int take(unsigned& n) const {
    const unsigned q = of(n), r = n - q * d;
    n = q;
    return (int)r;
  }
};

inline Divisor divisor(long long d) {
  Divisor v{(uint32_t)(d < 1 ? 1 : d), 0, 0};
  while ((1LL << v.shift) < (long long)v.d) ++v.shift;
  v.inverse = (uint32_t)((1ULL << (31 + v.shift)) / v.d + 1);
  return v;
}

}  // namespace rw
