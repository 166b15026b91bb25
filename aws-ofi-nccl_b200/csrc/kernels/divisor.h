// Division by a number that a launch knows.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

// floor(n / d) = floor(n m / 2^(32 + s)) for 0 <= n < 2^31, with 2^s < d <= 2^(s + 1) and m the least integer from 2^(32 + s) / d on: m d is beyond
// 2^(32 + s) by less than d, which times n is less than 2^(32 + s) (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994).
struct Divisor {
  int d = 1;
  uint32_t m = 0;
  int s = -1;   // -1: d is one
  Divisor() = default;
  explicit Divisor(int by) : d(by) {
    if (by == 1) return;
    s = 0;
    while ((1ll << (s + 1)) < by) ++s;
    m = static_cast<uint32_t>(((1ull << (32 + s)) + by - 1) / by);
  }
  __host__ __device__ __forceinline__ int quotient(int n) const {
#ifdef __CUDA_ARCH__
    return s < 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), m) >> s);
#else
    return s < 0 ? n : static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(n)) * m >> 32 >> s);
#endif
  }
};

}  // namespace b200
