// Division by a number that the host knows.
#pragma once

#include <cstdint>

namespace qw {

// x / d for 0 <= x < 2^31 by a product: q = (x + floor(x m / 2^32)) >> s with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d)
// + 1 (Granlund and Montgomery, 1994). The compiler's own division takes ten times the instructions, and the cache's kernels
// divide by the head group for every row and by the block size for every tile and token.
struct Divisor {
  uint32_t d, m, s;
  Divisor() = default;
  explicit Divisor(uint32_t of) : d(of), s(0) {
    while ((uint64_t{1} << s) < d) ++s;
    m = static_cast<uint32_t>((uint64_t{1} << 32) * ((uint64_t{1} << s) - d) / d + 1);
  }
  __device__ __forceinline__ int quotient(int x) const {
    return static_cast<int>((__umulhi(m, static_cast<uint32_t>(x)) + static_cast<uint32_t>(x)) >> s);
  }
  __device__ __forceinline__ int remainder(int x, int q) const { return x - q * static_cast<int>(d); }
};

}  // namespace qw
