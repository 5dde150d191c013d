// Quotients of kernel indices by numbers fixed per launch.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace nb {

// Quotients by a number that is fixed for a launch: n / d for 0 <= n < 2^31 as
// a high product and a shift (m = ceil(2^(32 + s) / d), s = ceil(log2 d) - 1,
// exact for 31-bit n because m * d - 2^(32 + s) < 2^(s + 1)).
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() : d(1), m(0), s(0) {}
  explicit FastDiv(uint32_t div) : d(div ? div : 1) {
    s = 0;
    while ((1ull << s) < d) ++s;  // ceil(log2 d)
    if (s == 0) {
      m = 0;  // d == 1
      return;
    }
    --s;
    m = (uint32_t)(((1ull << (32 + s)) + d - 1) / d);
  }
  __device__ __forceinline__ int div(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, m) >> s); }
};

}  // namespace nb
