// The positional mask's runs and vectors (kernels/positions.cuh) against its definition, by brute force.
#include <cstdio>
#include <initializer_list>

#include "kernels/positions.cuh"

int main() {
  long checked = 0;
  for (int keys = 1; keys <= 41; keys += 4)
    for (int window : {0, 1, 2, 7, 8, 9, 16, 40, 100})
      for (int sinks : {0, 1, 4, 8, 9, 30, 60})
        for (int p = -3; p < 60; ++p) {
          const cs::Visible v = cs::visible_keys(p, keys, window, sinks);
          const cs::VisibleVectors m = cs::visible_vectors(v);
          if (!(0 <= v.s_end && v.s_end <= v.lo && v.lo <= v.hi && v.hi <= keys)) return std::printf("runs %d %d %d %d\n", p, keys, window, sinks), 1;
          if (p >= 0) {
            const cs::Visible u = cs::visible_columns(p, keys, window, sinks);
            if (u.s_end != v.s_end || u.lo != v.lo || u.hi != v.hi) return std::printf("columns %d %d %d %d\n", p, keys, window, sinks), 1;
          }
          bool held[16] = {};
          for (int j = 0; j < m.n; ++j) {
            const int vec = cs::vector_at(m, j);
            if (vec < 0 || vec * 8 >= keys || held[vec]) return std::printf("vector %d %d %d %d\n", p, keys, window, sinks), 1;
            held[vec] = true;
          }
          for (int k = 0; k < keys; ++k) {
            const bool want = k <= p && (window == 0 || p - k < window || k < sinks);
            if (cs::sees(v, k) != want) return std::printf("sees %d %d %d %d key %d\n", p, keys, window, sinks, k), 1;
            if (((cs::visible_bits(v, k & ~7) >> (k & 7)) & 1) != (want ? 1u : 0u)) return std::printf("bits %d %d %d %d key %d\n", p, keys, window, sinks, k), 1;
            if (want && !held[k / 8]) return std::printf("not held %d %d %d %d key %d\n", p, keys, window, sinks, k), 1;
            ++checked;
          }
        }
  cs::Visible far = cs::visible_keys(2147483646, 2147483647, 16, 4);
  const cs::Visible same = cs::visible_columns(2147483646, 2147483647, 16, 4), all = cs::visible_columns(0, 5, 2147483647, 1);
  if (same.hi != far.hi || same.lo != far.lo || same.s_end != far.s_end || all.lo != 0 || all.hi != 1) return std::printf("columns far\n"), 1;
  if (far.hi != 2147483647 || far.lo != 2147483631 || far.s_end != 4) return std::printf("far\n"), 1;
  std::printf("ok %ld\n", checked);
  return 0;
}
