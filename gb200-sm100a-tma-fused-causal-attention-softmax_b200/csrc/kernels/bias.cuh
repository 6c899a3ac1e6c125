// Causal softmax with a learned relative-position bias, and its gradient.
//
// A group of 4 to 256 lanes works on one row at a time. The row's visible 16-byte
// vectors are copied to shared memory (cp.async) while the group works on the
// row before (long rows: once it is done with it), and the passes (maximum, sum,
// result; backward: the row's sum of p dp, result) read them there, so HBM sees
// each score once. Rows too long for that are read from global memory in each pass.
// Bound: HBM (2 bytes in per visible score, 2 out per column; the backward
// reads two matrices). B200, through the entry points in a stream, after a rest / in a
// second of calls, whose power holds the clock down: forward 64 x 4096^2 538 / 558 us,
// 0.92 / 0.88 of the copy rate; backward 32 x 4096^2 377 / 378 us, 0.87, 512 x 4096^2 5.7
// / 5.9 ms, 0.93 / 0.89; rows of 512 columns, bound by their instructions, 0.65 and 0.69.
//
// Bias: a distance d = position - key lies in the last bucket from its start
// on; the other distances (at most CS_MAX_BUCKET_START) are looked up in a
// shared-memory table of the head's bias by distance, in units of log2. Most
// vectors of a long row lie wholly in the last bucket and are wholly visible:
// these "plain" vectors take one constant, packed arithmetic and, for the
// maximum, a packed 16-bit comparison (scale >= 0 keeps the order); only the
// others pay for masks and look-ups. With both kinds in one unrolled loop over
// registers the instructions, not HBM, bound the kernel: 64 x 4096^2 took
// 1.0-2.5 ms at every split tried.
//
// Exponents are scale x + bias rounded once, minus the rounded maximum: fusing
// the subtraction into the multiply-add would leave the rounding error of the
// maximum, which a large scale blows up.
//
// A row whose maximum is kNarrow or more in magnitude leaves these fp32 exponents:
// their rounding would be a hundredth of a unit and more, and a finite score next to
// the type's ends (its lowest value as a mask) times log2 e is infinite. wide_row works
// such rows out in binary64, relative to the row's largest score; by their scores, fp16
// rows at a scale of up to 1 never are.
//
// Table gradient: a row holds each distance once, so a group adds its row's dz
// into its own array by distance without conflicts, row after row: no atomics,
// and the sums come in a fixed order. Distances in the last bucket go to a
// register per lane. Arrays, then CTAs, are summed in fixed order afterwards.
#pragma once

#include "common.cuh"
#include "divider.cuh"
#include "positions.cuh"
#include "types.cuh"

namespace cs {

constexpr int kMaxBuckets = 128;
constexpr int kBiasThreads = 128;     // CTA size while a row takes at most 4 warps
constexpr int kBiasMaxThreads = 256;  // rows of 8 warps
constexpr float kNarrow = 131072.f;   // 2^17, in units of log2

struct BiasParams {
  const uint16_t* x;    // scores; backward: probabilities
  const uint16_t* dp;   // backward: their gradient
  uint16_t* out;        // probabilities; backward: gradient of the scores
  const float* table;   // [heads, buckets]
  float* partial;       // backward: [matrix, CTA, buckets]
  int32_t heads, rows, cols, pitch, row_offset, window, sinks;
  int32_t ctas;         // per matrix
  int32_t lanes;        // of a group: a power of two, 4 to 256
  int32_t slots;        // vectors of one shared-memory row buffer (0: rows stay in global memory)
  int32_t buckets, near;  // near: first distance of the last bucket
  float scale;
  int32_t starts[kMaxBuckets];
};

// Arrays by distance hold 9 words per 8 distances, so that the lanes of a warp,
// 8 distances apart, meet different banks. A vector's distances d0, d0 - 1, ...
// d0 - 7 reach from -7 (masked) to near + 7 (clipped).
__host__ __device__ __forceinline__ int bias_slot(int d) { return d + 8 + ((d + 8) >> 3); }
__host__ __device__ __forceinline__ int bias_slots(int near) { return bias_slot(near + 7) + 1; }

__device__ __forceinline__ int bucket_of(const BiasParams& p, int d) {
  int lo = 0, hi = p.buckets;  // starts[lo] <= d < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.starts[mid] <= d) lo = mid; else hi = mid;
  }
  return lo;
}

// One group: its lanes, and what they do together. Groups of up to 32 lanes
// share a warp; larger ones take whole warps, a named barrier and a word of
// shared memory per warp.
struct Group {
  int lanes, id, rank;  // rank: this lane's
  uint32_t mask;        // the group's lanes of this warp
  __device__ __forceinline__ explicit Group(int n) : lanes(n) {
    id = threadIdx.x / n;
    rank = threadIdx.x - id * n;
    mask = n >= 32 ? 0xffffffffu : ((1u << n) - 1u) << (threadIdx.x & 31 & ~(n - 1));
  }
  __device__ __forceinline__ void sync() const {
    // Barriers by number: with a number in a register the kernel would get all 16 of
    // them, and the SM's 64 would hold it to four CTAs.
    if (lanes <= 32) __syncwarp(mask);
    else if (id == 0) asm volatile("bar.sync 1, %0;" ::"r"(lanes) : "memory");
    else asm volatile("bar.sync 2, %0;" ::"r"(lanes) : "memory");
  }
  __device__ __forceinline__ float max(float v, float* words) const {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, %2;" : "=f"(m) : "f"(v), "r"(mask));
    if (lanes > 32) {
      if ((rank & 31) == 0) words[rank >> 5] = m;
      sync();
      for (int k = 0; k < lanes >> 5; ++k) m = fmaxf(m, words[k]);
    }
    return m;
  }
  // The same for binary64 and any operation; words: two per warp. Its own barriers
  // keep the words from other uses, before and after.
  template <typename Op>
  __device__ __forceinline__ double join(double v, float* words, Op op) const {
    for (int o = (lanes < 32 ? lanes : 32) >> 1; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(mask, v, o));
    if (lanes > 32) {
      sync();
      if ((rank & 31) == 0) {
        words[rank >> 4] = __int_as_float(__double2hiint(v));
        words[(rank >> 4) + 1] = __int_as_float(__double2loint(v));
      }
      sync();
      v = __hiloint2double(__float_as_int(words[0]), __float_as_int(words[1]));
      for (int k = 1; k < lanes >> 5; ++k)
        v = op(v, __hiloint2double(__float_as_int(words[2 * k]), __float_as_int(words[2 * k + 1])));
      sync();
    }
    return v;
  }
  __device__ __forceinline__ float sum(float v, float* words) const {
    for (int o = (lanes < 32 ? lanes : 32) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    if (lanes > 32) {
      if ((rank & 31) == 0) words[rank >> 5] = v;
      sync();
      v = 0.f;
      for (int k = 0; k < lanes >> 5; ++k) v += words[k];
    }
    return v;
  }
};

// One row: its visible vectors, numbered densely, and the plain ones among
// them, [f0, f1): wholly visible and wholly in the last bucket.
struct RowWalk {
  Visible v;
  VisibleVectors m;
  int32_t pos, f0, f1;
  __device__ __forceinline__ RowWalk(const BiasParams& p, int row) {
    pos = p.row_offset + row;  // below 2^31
    v = visible_columns(pos, p.cols, p.window, p.sinks);
    m = visible_vectors(v);
    f0 = m.n_sink + ((v.lo & 7) ? 1 : 0);
    // Last element 8 j + 7 of window vector j: below hi and at distance near or more.
    const int32_t end = min(v.hi, pos - p.near + 1) >> 3;
    f1 = max(f0, min(m.n, m.n_sink + end - m.w_beg));
    if (v.lo >= v.hi) f0 = f1 = m.n;
  }
  // The vectors that are not plain, numbered densely.
  __device__ __forceinline__ int others() const { return m.n - (f1 - f0); }
  __device__ __forceinline__ int other(int t) const { return t < f0 ? t : t - f0 + f1; }
};

__device__ __forceinline__ void zero_masked(const BiasParams& p, const RowWalk& w, uint4* row, int gt, int gn) {
  const uint4 z = make_uint4(0, 0, 0, 0);
  const int w_end = w.m.w_beg + w.m.n - w.m.n_sink;
  for (int j = w.m.n_sink + gt; j < w.m.w_beg; j += gn) __stcs(row + j, z);
  for (int j = w_end + gt; j < (p.pitch >> 3); j += gn) __stcs(row + j, z);
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void fetch_row(const RowWalk& w, const uint4* in, uint4* buffer, int gt, int gn) {
  for (int j = gt; j < w.m.n; j += gn) cp_async16(buffer + j, in + vector_at(w.m, j));
}

template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& r, F2* f) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 t = T::unpack(w[q]);
    f[q] = f2(t.x, t.y);
  }
}

// 2^(scale x + bias - m) of a plain vector.
template <typename T>
__device__ __forceinline__ void plain_exp(const uint4& raw, F2 sl, F2 far, F2 minus_m, F2* e) {
  unpack_pairs<T>(raw, e);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 t = f2_out(f2_add(f2_fma(e[q], sl, far), minus_m));
    e[q] = f2(ex2(t.x), ex2(t.y));
  }
}

// Slots of a vector's distances: that of element e is first - e - (e > part).
struct DistanceSlots {
  int first, part;
  __device__ __forceinline__ DistanceSlots(int d0, int near) {
    const int d = min(d0, near + 7);  // all 8 are in the last bucket from there on
    first = bias_slot(d);
    part = d & 7;
  }
  __device__ __forceinline__ int operator[](int e) const { return first - e - (e > part ? 1 : 0); }
};

// The biased scores of any vector in units of log2; -infinity where masked.
template <typename T>
__device__ __forceinline__ uint32_t biased8(const BiasParams& p, const RowWalk& w, const float* tab, float sl, int c0,
                                            const uint4& raw, float* z) {
  unpack8<T>(raw, z);
  const uint32_t bits = visible_bits(w.v, c0);
  const DistanceSlots at(w.pos - c0, p.near);
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] = (bits >> e) & 1 ? __fmaf_rn(z[e], sl, tab[at[e]]) : -INFINITY;
  return bits;
}

__device__ __forceinline__ float max8(const float* z) {
  return fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7])));
}

__device__ __forceinline__ float sum8(const float* z) {
  return ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7]));
}

// A row in binary64: scale (x - top) + bias, top the largest score seen, so that
// neither overflows and the bias counts beside scores of any size. A lane takes one
// column at a time. table: the head's.
template <typename T>
__device__ __forceinline__ void wide_row(const BiasParams& p, const RowWalk& w, const Group& group, const uint16_t* from,
                                         const float* table, float* words, uint16_t* out) {
  constexpr double kInfinity = INFINITY, kLog2 = 1.4426950408889634;
  auto larger = [](double a, double b) { return fmax(a, b); };
  // f(column, score, whether it is seen) of this lane's columns among the visible vectors.
  auto each = [&](auto f) {
#pragma unroll 1
    for (uint32_t i = group.rank; i < (uint32_t)w.m.n * 8u; i += group.lanes) {
      const int at = vector_at(w.m, i >> 3) * 8, e = i & 7;
      f(at + e, T::unpack(from[at + e]).x, ((visible_bits(w.v, at) >> e) & 1) != 0);
    }
  };
  // The largest score; +infinity if one is a NaN: on to the sum.
  float most = -INFINITY;
  for (int j = group.rank; j < w.m.n; j += group.lanes) {
    const int at = vector_at(w.m, j) * 8;
    float x[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(from + at), x);
    const uint32_t bits = visible_bits(w.v, at);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((bits >> e) & 1) most = fmaxf(most, x[e] == x[e] ? x[e] : INFINITY);
  }
  double top = group.join(most, words, larger);
  if (top == -kInfinity) {  // all of them -infinity
    for (int j = group.rank; j < w.m.n; j += group.lanes)
      *reinterpret_cast<uint4*>(out + vector_at(w.m, j) * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  if (top == kInfinity) top = 0.0;
  const double last = table[p.buckets - 1];
  auto score = [&](int c, float x) {
    const int d = w.pos - c;
    return (double)p.scale * ((double)x - top) + (d >= p.near ? last : (double)table[bucket_of(p, d)]);
  };
  double m = -kInfinity, s = 0.0;
  each([&](int c, float x, bool seen) {
    if (seen) m = fmax(m, score(c, x));
  });
  m = group.join(m, words, larger);
  if (m == -kInfinity) m = 0.0;  // by the bias: every exponential is 0
  each([&](int c, float x, bool seen) {
    if (seen) s += ex2((float)((score(c, x) - m) * kLog2));
  });
  s = group.join(s, words, [](double a, double b) { return a + b; });
  const float inv = s == 0.0 ? 0.f : rcp_rn((float)s);  // a NaN stays one
  each([&](int c, float x, bool seen) {
    out[c] = seen ? (uint16_t)T::pack(ex2((float)((score(c, x) - m) * kLog2)) * inv, 0.f) : (uint16_t)0;
  });
}

// A warp's wide rows once more: the marked ones, or all of them. (Kept apart from the
// main loop, which pays for a register more or a call in it with every row: rows of
// 512 columns bf16 188 us, 195 to 219.)
template <typename T>
__device__ __forceinline__ void wide_rows(const BiasParams& p, float* words, bool all) {
  const Group group(p.lanes);
  const int groups = blockDim.x / p.lanes;
  const int64_t matrix = blockIdx.x / p.ctas;
  const int cta = blockIdx.x - (int)(matrix * p.ctas);
  words += (threadIdx.x / 32 - group.rank / 32) * 2;
  group.sync();  // the other warps' marks
  for (RowTurns turns(p.rows, cta * groups + group.id, p.ctas * groups); turns.inside(); turns.next()) {
    const RowWalk w(p, turns.here());
    if (w.m.n == 0) continue;
    const int64_t row = (matrix * p.rows + turns.here()) * p.pitch;
    uint16_t* out = p.out + row;
    const float mark = T::unpack(out[w.v.s_end > 0 ? 0 : w.v.lo]).x;
    group.sync();  // all have read it
    if (all || mark != mark) wide_row<T>(p, w, group, p.x + row, p.table + (matrix % p.heads) * p.buckets, words, out);
  }
}

// kBuffers: of a group in shared memory, p.slots vectors each; 0: rows stay in global memory.
template <typename T, int kBuffers>
__global__ void __launch_bounds__(kBiasMaxThreads) bias_softmax_kernel(const __grid_constant__ BiasParams p) {
  constexpr bool kStaged = kBuffers > 0;
  extern __shared__ __align__(16) uint4 smem[];
  const Group group(p.lanes);
  const int gn = p.lanes, groups = blockDim.x / gn, gt = group.rank;
  uint4* buffers = smem + group.id * kBuffers * p.slots;
  float* tab = reinterpret_cast<float*>(smem + groups * kBuffers * p.slots);  // bias by distance, [0, near]
  float* words = tab + bias_slots(p.near);  // two per warp, for groups of several warps
  // Whether this warp met wide rows; whether all rows are.
  int* wide = reinterpret_cast<int*>(words + (blockDim.x / 32 + threadIdx.x / 32) * 2);
  float* words_max = words + (threadIdx.x / 32 - gt / 32) * 2;
  float* words_sum = words_max + (gn >> 5);
  const int64_t matrix = blockIdx.x / p.ctas;
  const int cta = blockIdx.x - (int)(matrix * p.ctas);
  const float* table = p.table + (matrix % p.heads) * p.buckets;
  const int64_t base = matrix * p.rows * (int64_t)p.pitch;
  RowTurns turns(p.rows, cta * groups + group.id, p.ctas * groups);

  pdl_wait();
  auto source = [&](int r) { return reinterpret_cast<const uint4*>(p.x + base + (int64_t)r * p.pitch); };
  if (kStaged) {
    if (turns.inside()) fetch_row(RowWalk(p, turns.row()), source(turns.row()), buffers, gt, gn);
    cp_async_commit();
  }
  bool large = false;
  for (int d = threadIdx.x - 8; d < p.near + 8; d += blockDim.x) {
    const float v = table[bucket_of(p, max(d, 0))], t = v * kLog2e;
    large |= t >= 0x1p126f;  // a score's sum with it may not fit
    tab[bias_slot(d)] = t < -0x1p127f ? -0x1p127f : t;  // a mask; rows of nothing else are wide
  }
  wide[0] = 0;
  wide[1] = __syncthreads_or(large);
  const float far = tab[bias_slot(p.near)], sl = p.scale * kLog2e;
  const F2 far2 = f2(far, far), sl2 = f2(sl, sl);

  RowWalk w(p, turns.row());
  for (int turn = 0; turns.inside(); turns.next(), turn ^= 1) {
    const int row = turns.here(), after = turns.next_row();
    uint4* out = reinterpret_cast<uint4*>(p.out + base + (int64_t)row * p.pitch);
    const uint4* in = source(row);
    const uint4* staged = buffers + (kBuffers == 2 ? turn * p.slots : 0);
    const RowWalk next(p, after);
    if (kBuffers == 2) {
      group.sync();  // the row before, in the other buffer, is done with
      if (!turns.last()) fetch_row(next, source(after), buffers + (turn ^ 1) * p.slots, gt, gn);
      cp_async_commit();
    }
    zero_masked(p, w, out, gt, gn);
    if (kStaged) {
      cp_async_wait<kBuffers == 2 ? 1 : 0>();
      group.sync();
    }
    auto vec = [&](int j) { return kStaged ? staged[j] : in[vector_at(w.m, j)]; };
    // A lane's first vector that is not plain, mostly its only one, stays in registers.
    const int others = w.others(), at0 = vector_at(w.m, w.other(gt));
    float z[8], z0[8];
    F2 e[4];
    uint32_t bits0 = 0;
    float m = -INFINITY;
    if (gt < others) {
      bits0 = biased8<T>(p, w, tab, sl, at0 * 8, vec(w.other(gt)), z0);
      m = max8(z0);
    }
    for (int t = gt + gn; t < others; t += gn) {
      const int j = w.other(t);
      biased8<T>(p, w, tab, sl, vector_at(w.m, j) * 8, vec(j), z);
      m = fmaxf(m, max8(z));
    }
    if (w.f0 + gt < w.f1) {
      uint32_t most = vector_max<T>(vec(w.f0 + gt));
#pragma unroll 4
      for (int j = w.f0 + gt + gn; j < w.f1; j += gn) most = T::max2(most, vector_max<T>(vec(j)));
      const float2 t = T::unpack(most);
      m = fmaxf(m, __fmaf_rn(fmaxf(t.x, t.y), sl, far));
    }
    m = fmaxf(group.max(m, words_max), -3.0e38f);  // a row of -infinity only: every exponential is 0
    const F2 minus_m = f2(-m, -m);

    float s = 0.f;
    F2 s2 = f2(0.f, 0.f), s3 = s2;
    if (gt < others) {
#pragma unroll
      for (int q = 0; q < 8; ++q) z0[q] = ex2(z0[q] - m);
      s = sum8(z0);
    }
    for (int t = gt + gn; t < others; t += gn) {
      const int j = w.other(t);
      biased8<T>(p, w, tab, sl, vector_at(w.m, j) * 8, vec(j), z);
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = ex2(z[q] - m);
      s += sum8(z);
    }
#pragma unroll 2
    for (int j = w.f0 + gt; j < w.f1; j += gn) {
      plain_exp<T>(vec(j), sl2, far2, minus_m, e);
      s2 = f2_add(s2, f2_add(e[0], e[1]));
      s3 = f2_add(s3, f2_add(e[2], e[3]));
    }
    const float2 s4 = f2_out(f2_add(s2, s3));
    s = group.sum(s + (s4.x + s4.y), words_sum);
    float inv = rcp_rn(s);  // s >= 1, or a NaN
    if (!(fabsf(m) < kNarrow)) {
      // Nothing but -infinity: so were the scores, if their multiples are finite. Else a
      // wide row, marked by NaN in all visible columns.
      inv = s == 0.f && (T::kIsHalf || p.scale <= 0.25f) ? 0.f : NAN;
      if (inv != 0.f) wide[0] = 1;
    }
    const F2 inv2 = f2(inv, inv);

    if (gt < others) {
#pragma unroll
      for (int q = 0; q < 8; ++q) z0[q] = (bits0 >> q) & 1 ? z0[q] * inv : 0.f;  // +0.0 in a NaN row too
      __stcs(out + at0, pack8<T>(z0));
    }
    for (int t = gt + gn; t < others; t += gn) {
      const int j = w.other(t), at = vector_at(w.m, j);
      const uint32_t bits = biased8<T>(p, w, tab, sl, at * 8, vec(j), z);
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = (bits >> q) & 1 ? ex2(z[q] - m) * inv : 0.f;
      __stcs(out + at, pack8<T>(z));
    }
    uint4* plain_out = out + (w.m.w_beg - w.m.n_sink);  // plain vectors are the window's
#pragma unroll 2
    for (int j = w.f0 + gt; j < w.f1; j += gn) {
      plain_exp<T>(vec(j), sl2, far2, minus_m, e);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 t = f2_out(f2_mul(e[q], inv2));
        z[2 * q] = t.x;
        z[2 * q + 1] = t.y;
      }
      __stcs(plain_out + j, pack8<T>(z));
    }
    if (kBuffers == 1) {
      group.sync();
      if (!turns.last()) fetch_row(next, source(after), buffers, gt, gn);
      cp_async_commit();
    }
    w = next;
  }
  __syncwarp();
  if (wide[0] || wide[1]) wide_rows<T>(p, words, wide[1] != 0);
  pdl_trigger();
}

template <typename T, int kBuffers>
__global__ void __launch_bounds__(kBiasMaxThreads) bias_backward_kernel(const __grid_constant__ BiasParams p) {
  constexpr bool kStaged = kBuffers > 0;
  extern __shared__ __align__(16) uint4 smem[];
  const Group group(p.lanes);
  const int gn = p.lanes, groups = blockDim.x / gn, gt = group.rank, lane = threadIdx.x & 31;
  const int slots = bias_slots(p.near);
  uint4* buffers = smem + group.id * 2 * kBuffers * p.slots;  // a row of p and one of dp each
  float* sums = reinterpret_cast<float*>(smem + groups * 2 * kBuffers * p.slots);
  float* acc = sums + group.id * slots;  // sums by distance, [0, near)
  float* words = sums + groups * slots + (threadIdx.x / 32 - gt / 32);  // one per warp
  float* far_sums = sums + groups * slots + blockDim.x / 32;  // one per warp
  const int64_t matrix = blockIdx.x / p.ctas;
  const int cta = blockIdx.x - (int)(matrix * p.ctas);
  const int64_t base = matrix * p.rows * (int64_t)p.pitch;
  RowTurns turns(p.rows, cta * groups + group.id, p.ctas * groups);
  for (int d = gt; d < slots; d += gn) acc[d] = 0.f;

  pdl_wait();
  auto source = [&](const uint16_t* x, int r) { return reinterpret_cast<const uint4*>(x + base + (int64_t)r * p.pitch); };
  auto fetch = [&](const RowWalk& w, int r, uint4* to) {
    fetch_row(w, source(p.x, r), to, gt, gn);
    fetch_row(w, source(p.dp, r), to + p.slots, gt, gn);
  };
  if (kStaged) {
    if (turns.inside()) fetch(RowWalk(p, turns.row()), turns.row(), buffers);
    cp_async_commit();
  }
  group.sync();
  float far = 0.f;

  RowWalk w(p, turns.row());
  for (int turn = 0; turns.inside(); turns.next(), turn ^= 1) {
    const int row = turns.here(), after = turns.next_row();
    uint4* out = reinterpret_cast<uint4*>(p.out + base + (int64_t)row * p.pitch);
    const uint4* in = source(p.x, row);
    const uint4* in2 = source(p.dp, row);
    const uint4* staged = buffers + (kBuffers == 2 ? turn * 2 * p.slots : 0);
    const RowWalk next(p, after);
    if (kBuffers != 1) group.sync();  // the row before is done with: its buffer, and its additions to acc
    if (kBuffers == 2) {
      if (!turns.last()) fetch(next, after, buffers + (turn ^ 1) * 2 * p.slots);
      cp_async_commit();
    }
    zero_masked(p, w, out, gt, gn);
    if (kStaged) {
      cp_async_wait<kBuffers == 2 ? 1 : 0>();
      group.sync();
    }
    auto vec = [&](int j) { return kStaged ? staged[j] : in[vector_at(w.m, j)]; };
    auto vec2 = [&](int j) { return kStaged ? staged[p.slots + j] : in2[vector_at(w.m, j)]; };
    const int others = w.others(), at0 = vector_at(w.m, w.other(gt));
    float a[8], g[8], a0[8], g0[8];
    F2 x[4], y[4];
    // p and dp of any vector, 0 where masked.
    auto masked8 = [&](int j, int at, float* a, float* g) {
      unpack8<T>(vec(j), a);
      unpack8<T>(vec2(j), g);
      const uint32_t bits = visible_bits(w.v, at * 8);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (!((bits >> q) & 1)) a[q] = g[q] = 0.f;
      return bits;
    };
    uint32_t bits0 = 0;
    float dot = 0.f;
    F2 d2 = f2(0.f, 0.f), d3 = d2;
    if (gt < others) {
      bits0 = masked8(w.other(gt), at0, a0, g0);
#pragma unroll
      for (int q = 0; q < 8; ++q) dot = __fmaf_rn(a0[q], g0[q], dot);
    }
    for (int t = gt + gn; t < others; t += gn) {
      const int j = w.other(t);
      masked8(j, vector_at(w.m, j), a, g);
#pragma unroll
      for (int q = 0; q < 8; ++q) dot = __fmaf_rn(a[q], g[q], dot);
    }
#pragma unroll 2
    for (int j = w.f0 + gt; j < w.f1; j += gn) {
      unpack_pairs<T>(vec(j), x);
      unpack_pairs<T>(vec2(j), y);
      d2 = f2_fma(x[0], y[0], d2);
      d3 = f2_fma(x[1], y[1], d3);
      d2 = f2_fma(x[2], y[2], d2);
      d3 = f2_fma(x[3], y[3], d3);
    }
    const float2 d4 = f2_out(f2_add(d2, d3));
    dot = group.sum(dot + (d4.x + d4.y), words);

    // Distances below 0 (masked) and from near on have slots of their own that
    // nothing reads or that count to the last bucket; clipped ones go to a register.
    auto finish8 = [&](int at, uint32_t bits, float* a, const float* g) {
      const int d0 = w.pos - at * 8;
      const DistanceSlots slot(d0, p.near);
#pragma unroll
      for (int q = 0; q < 8; ++q) a[q] = (bits >> q) & 1 ? a[q] * (g[q] - dot) : 0.f;  // masked: 0 in a NaN row too
      if (d0 > p.near + 7) {
        far += sum8(a);
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[slot[q]] += a[q];
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) a[q] *= p.scale;
      __stcs(out + at, pack8<T>(a));
    };
    if (gt < others) finish8(at0, bits0, a0, g0);
    for (int t = gt + gn; t < others; t += gn) {
      const int j = w.other(t), at = vector_at(w.m, j);
      const uint32_t bits = masked8(j, at, a, g);
      finish8(at, bits, a, g);
    }
    uint4* plain_out = out + (w.m.w_beg - w.m.n_sink);
    const F2 minus_dot = f2(-dot, -dot), scale2 = f2(p.scale, p.scale);
    F2 far2 = f2(0.f, 0.f);
#pragma unroll 2
    for (int j = w.f0 + gt; j < w.f1; j += gn) {
      unpack_pairs<T>(vec(j), x);
      unpack_pairs<T>(vec2(j), y);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = f2_mul(x[q], f2_add(y[q], minus_dot));
      far2 = f2_add(far2, f2_add(f2_add(x[0], x[1]), f2_add(x[2], x[3])));
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 t = f2_out(f2_mul(x[q], scale2));
        a[2 * q] = t.x;
        a[2 * q + 1] = t.y;
      }
      __stcs(plain_out + j, pack8<T>(a));
    }
    const float2 far3 = f2_out(far2);
    far += far3.x + far3.y;
    if (kBuffers == 1) {
      group.sync();
      if (!turns.last()) fetch(next, after, buffers);
      cp_async_commit();
    }
    w = next;
  }
  far = warp_sum(far);
  if (lane == 0) far_sums[threadIdx.x >> 5] = far;
  __syncthreads();
  // The groups' arrays into the first, then 8 lanes a bucket. (A warp a bucket, over all
  // groups' arrays: 72 x 72^2 26.4 us, this 7.8; 132 x 1085^2 208, 176.)
  for (int d = threadIdx.x; d < slots; d += blockDim.x) {
    float s = sums[d];
#pragma unroll 8
    for (int k = 1; k < groups; ++k) s += sums[k * slots + d];
    sums[d] = s;
  }
  __syncthreads();
  float* partial = p.partial + (int64_t)blockIdx.x * p.buckets;
  const int part = threadIdx.x & 7;
  for (int b0 = 0; b0 < p.buckets; b0 += blockDim.x / 8) {
    const int b = b0 + (threadIdx.x >> 3);
    float s = 0.f;
    if (b == p.buckets - 1) {
      s = sums[bias_slot(p.near + part)] + (part < (int)(blockDim.x / 32) ? far_sums[part] : 0.f);
    } else if (b < p.buckets) {
      for (int d = p.starts[b] + part; d < p.starts[b + 1]; d += 8) s += sums[bias_slot(d)];
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (part == 0 && b < p.buckets) partial[b] = s;
  }
  pdl_trigger();
}

struct BiasReduceParams {
  const float* partial;
  float* dtable;
  int32_t batch, heads, ctas, buckets;
  Divider by_ctas;
};

// dtable[h, j]: grid.x heads, grid.y tiles of 32 buckets. Lanes are buckets, so
// that a warp's loads are contiguous; the warps take turns at the partials and
// their sums are added in a fixed order, in 64 bits.
__global__ void __launch_bounds__(1024) bias_table_kernel(const __grid_constant__ BiasReduceParams p) {
  __shared__ double sums[32][33];
  pdl_wait();
  const int h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.y * 32 + lane;
  double s = 0.0;
  if (b < p.buckets) {
    // CTAs of the head's matrices, one after the other.
    const int n = p.batch * p.ctas;
#pragma unroll 8
    for (int c = warp; c < n; c += 32) {
      const int k = p.by_ctas.div(c);
      s += (double)p.partial[(((int64_t)k * p.heads + h) * p.ctas + (c - k * p.ctas)) * p.buckets + b];
    }
  }
  sums[warp][lane] = s;
  __syncthreads();
  double t = sums[lane][warp];  // warp: the bucket, lane: whose sum
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int bucket = blockIdx.y * 32 + warp;
  if (lane == 0 && bucket < p.buckets) p.dtable[(int64_t)h * p.buckets + bucket] = (float)t;
}

}  // namespace cs
