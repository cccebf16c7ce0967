// Division of 0 <= n < 2^31 by a fixed 1 <= d < 2^31 as a multiplication and a
// shift.  With s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1 the quotient
// is (hi32(m n) + n) >> s: hi32(m n) <= n, so the sum stays below 2^32, and
// (2^32 + m) / 2^(32 + s) exceeds 1 / d by less than 1 / (2^31 d) for such n.
#pragma once
#include <cstdint>

namespace bw {

struct FastDiv {
  uint32_t d = 1, m = 1, s = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((uint64_t(1) << s) < div) ++s;
    m = (uint32_t)((((uint64_t(1) << s) - div) << 32) / div) + 1;
  }
#ifdef __CUDACC__
  __host__ __device__
#endif
  uint32_t div(uint32_t n) const {
#ifdef __CUDA_ARCH__
    return (__umulhi(m, n) + n) >> s;
#else
    return (uint32_t)((((uint64_t)m * n) >> 32) + n) >> s;
#endif
  }
};

}  // namespace bw
