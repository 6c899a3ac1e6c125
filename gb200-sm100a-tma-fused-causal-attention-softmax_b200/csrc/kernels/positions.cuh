// The positional mask shared by the biased softmax and the attention kernels.
//
// A query at absolute position p sees key k when
//     k <= p  and  k < keys  and  (window == 0 or p - k < window or k < sinks).
// So a row's visible keys are at most two runs: [0, s_end) and [lo, hi) with
// s_end <= lo. Plain integer code, host-callable: the CPU tests compile it as C++.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define CS_HD __host__ __device__ __forceinline__
#else
#define CS_HD inline
#endif

namespace cs {

struct Visible {
  int32_t s_end;   // sinks: [0, s_end)
  int32_t lo, hi;  // the window: [lo, hi), empty if lo >= hi
};

// window > 0, or 0 for none. p may be negative (a query before the first key: sees nothing).
CS_HD Visible visible_keys(int64_t p, int32_t keys, int32_t window, int32_t sinks) {
  Visible v;
  const int64_t hi = p + 1 < keys ? p + 1 : keys;
  v.hi = (int32_t)(hi > 0 ? hi : 0);
  const int64_t lo = window > 0 ? p + 1 - window : 0;
  const int64_t lo0 = lo > 0 ? lo : 0;
  const int32_t cut = (int32_t)(lo0 < v.hi ? lo0 : v.hi);
  v.lo = cut;  // lo == hi for an empty window run
  v.s_end = sinks < cut ? sinks : cut;
  return v;
}

// The same for 0 <= p <= 2^31 - 2 in 32-bit arithmetic.
CS_HD Visible visible_columns(int32_t p, int32_t keys, int32_t window, int32_t sinks) {
  Visible v;
  v.hi = p + 1 < keys ? p + 1 : keys;
  const int32_t lo = window > 0 ? p + 1 - window : 0;
  const int32_t lo0 = lo > 0 ? lo : 0;
  v.lo = lo0 < v.hi ? lo0 : v.hi;
  v.s_end = sinks < v.lo ? sinks : v.lo;
  return v;
}

CS_HD bool sees(const Visible& v, int32_t k) { return k < v.s_end || (k >= v.lo && k < v.hi); }

// The 8-element vectors that hold a row's visible columns, numbered densely:
// vector j < n_sink is vector j of the row, the others start at w_beg.
struct VisibleVectors {
  int32_t n_sink, w_beg, n;
};

CS_HD VisibleVectors visible_vectors(const Visible& v) {
  VisibleVectors m;
  const int32_t s_vec = (v.s_end + 7) >> 3;
  const int32_t w_beg = v.lo < v.hi ? v.lo >> 3 : s_vec;
  const int32_t w_end = v.lo < v.hi ? (v.hi + 7) >> 3 : s_vec;
  m.n_sink = s_vec < w_beg ? s_vec : w_beg;
  m.w_beg = w_beg;
  m.n = m.n_sink + (w_end - w_beg);
  return m;
}

CS_HD int32_t clip8(int32_t n) { return n < 0 ? 0 : n > 8 ? 8 : n; }

// Bit e: the row sees column c0 + e.
CS_HD uint32_t visible_bits(const Visible& v, int32_t c0) {
  const uint32_t below_hi = (1u << clip8(v.hi - c0)) - 1u, below_lo = (1u << clip8(v.lo - c0)) - 1u;
  return (below_hi & ~below_lo) | ((1u << clip8(v.s_end - c0)) - 1u);
}

CS_HD int32_t vector_at(const VisibleVectors& m, int32_t j) { return j < m.n_sink ? j : j - m.n_sink + m.w_beg; }

// The rows that one of a matrix's groups of lanes takes in turn, the last (longest)
// ones first: row rows - 1 - i for i = first, first + step, ... In unsigned
// arithmetic: i + step passes 2^31 - 1 where rows is close to it. 0 <= first, step <
// 2^31. (Counted down in signed numbers: backward 32 x 4096^2 377 us, this 371.)
struct RowTurns {
  uint32_t i, step, rows;
  CS_HD RowTurns(int32_t rows, int32_t first, int32_t step) : i((uint32_t)first), step((uint32_t)step), rows((uint32_t)rows) {}
  CS_HD bool inside() const { return i < rows; }
  CS_HD bool last() const { return i + step >= rows; }
  CS_HD int32_t here() const { return (int32_t)(rows - 1 - i); }  // inside only
  CS_HD int32_t row() const { return i < rows ? here() : 0; }     // 0: read ahead, not used
  CS_HD int32_t next_row() const { return i + step < rows ? (int32_t)(rows - 1 - i - step) : 0; }
  CS_HD void next() { i += step; }
};

}  // namespace cs
