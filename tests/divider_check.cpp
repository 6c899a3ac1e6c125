// Division by a host-known number (kernels/divider.cuh) against the machine's.
#include <cstdio>
#include <initializer_list>

#include "kernels/divider.cuh"

int main() {
  const uint32_t top = 2147483647u;
  long checked = 0;
  auto check = [&](uint32_t d, uint32_t n) {
    const cs::Divider by = cs::Divider::of(d);
    ++checked;
    if ((uint32_t)by.div((int)n) == n / d && (uint32_t)by.mod((int)n) == n % d) return true;
    std::printf("%u / %u\n", n, d);
    return false;
  };
  uint32_t seed = 1;
  auto any = [&] { return (seed = seed * 1664525u + 1013904223u) >> 1; };
  for (uint32_t i = 0; i < 70000; ++i) {
    // Small divisors, those next to powers of two, the largest, any.
    const uint32_t ds[] = {i + 1, (1u << (i % 31)) + i % 3, (1u << (1 + i % 30)) - 1, top - i, any() >> (i % 31)};
    for (uint32_t d : ds) {
      if (d == 0 || d > top) continue;
      const uint32_t most = top / d * d;
      for (uint32_t n : {0u, d - 1, d, most - 1, most, top, any(), any() / d * d})
        if (!check(d, n)) return 1;
    }
  }
  std::printf("ok %ld\n", checked);
  return 0;
}
