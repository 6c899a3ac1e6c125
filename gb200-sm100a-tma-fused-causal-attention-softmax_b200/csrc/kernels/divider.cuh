// Division by a number that the host knows.
#pragma once

#include "positions.cuh"

namespace cs {

// Division by a number the host knows, for 0 <= n < 2^31: a CTA of a few tiles
// would spend a tenth of its time on the compiler's division routine.
struct Divider {
  uint32_t by, mul, shift;
  static Divider of(uint32_t d) {  // 1 <= d < 2^31
    Divider r{d, 0, 31};
    while ((1ull << (r.shift - 31)) < d) ++r.shift;
    r.mul = (uint32_t)(((1ull << r.shift) + d - 1) / d);
    return r;
  }
  CS_HD int div(int n) const { return (int)((uint64_t)(uint32_t)n * mul >> shift); }
  CS_HD int mod(int n) const { return n - div(n) * (int)by; }
};

}  // namespace cs
