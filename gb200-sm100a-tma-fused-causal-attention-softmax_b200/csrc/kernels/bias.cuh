// Causal softmax with a learned relative-position bias, and its gradient.
//
// A group of W warps owns one row at a time; each lane keeps V 16-byte vectors
// of the row's visible columns in registers, so scores (or probabilities and
// their gradients) are read once. Rows longer than the group's registers are
// walked in chunks and read again from L2. Bound: HBM (2 bytes in per visible
// score, 2 out per column; the backward reads two matrices).
//
// Bias: a distance d = position - key lies in the last bucket from its start
// on, and the other distances (fewer than CS_MAX_BUCKET_START) are looked up in
// a shared-memory table of the head's bias by distance, already in units of
// log2. Vectors wholly in the last bucket, most of a long row, take one constant.
//
// Table gradient: a row holds each distance once, so a group adds its row's dz
// into its own array by distance without conflicts, row after row: no atomics,
// and the sums come in a fixed order. Distances in the last bucket go to a
// register per lane. Arrays, then CTAs, are summed in fixed order afterwards.
#pragma once

#include "common.cuh"
#include "positions.cuh"
#include "types.cuh"

namespace cs {

constexpr int kMaxBuckets = 128;
constexpr int kBiasThreads = 256;     // CTA size while a row takes at most 8 warps
constexpr int kBiasMaxThreads = 512;  // CTA size of longer rows (16 warps a row)

struct BiasParams {
  const uint16_t* x;    // scores; backward: probabilities
  const uint16_t* dp;   // backward: their gradient
  uint16_t* out;        // probabilities; backward: gradient of the scores
  const float* table;   // [heads, buckets]
  float* partial;       // backward: [matrix, CTA, buckets]
  int32_t heads, rows, cols, pitch, row_offset, window, sinks;
  int32_t ctas;         // per matrix
  int32_t warps;        // W, per row
  int32_t buckets, near;  // near: first distance of the last bucket
  float scale;
  int32_t starts[kMaxBuckets];
};

// Distances sit 9 words per 8, so that the lanes of a warp, 8 distances apart,
// meet different banks.
__host__ __device__ __forceinline__ int bias_slot(int d) { return d + (d >> 3); }

__device__ __forceinline__ int bucket_of(const BiasParams& p, int d) {
  int lo = 0, hi = p.buckets;  // starts[lo] <= d < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.starts[mid] <= d) lo = mid; else hi = mid;
  }
  return lo;
}

// Barrier of one group's threads (W warps; one warp needs none).
__device__ __forceinline__ void group_sync(int id, int threads) {
  if (threads == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

struct RowWalk {
  Visible v;
  VisibleVectors m;
  int32_t pos;
  __device__ __forceinline__ RowWalk(const BiasParams& p, int row) {
    const int64_t at = (int64_t)p.row_offset + row;
    v = visible_keys(at, p.cols, p.window, p.sinks);
    m = visible_vectors(v);
    pos = (int32_t)at;
  }
};

__device__ __forceinline__ void zero_masked(const BiasParams& p, const RowWalk& w, uint4* row, int gt, int gn) {
  const uint4 z = make_uint4(0, 0, 0, 0);
  const int w_end = w.m.w_beg + w.m.n - w.m.n_sink;
  for (int j = w.m.n_sink + gt; j < w.m.w_beg; j += gn) __stcs(row + j, z);
  for (int j = w_end + gt; j < (p.pitch >> 3); j += gn) __stcs(row + j, z);
}

// The biased scores of one vector in units of log2; -infinity where masked.
template <typename T>
__device__ __forceinline__ void biased8(const BiasParams& p, const RowWalk& w, const float* tab, float far, float sl,
                                        int c0, const uint4& raw, float* z) {
  unpack8<T>(raw, z);
  const int d0 = w.pos - c0;
  if (d0 - 7 >= p.near) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = __fmaf_rn(z[e], sl, far);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = min(max(d0 - e, 0), p.near);
      z[e] = __fmaf_rn(z[e], sl, tab[bias_slot(d)]);
    }
  }
  if (!((c0 >= w.v.lo && c0 + 8 <= w.v.hi) || c0 + 8 <= w.v.s_end)) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!sees(w.v, c0 + e)) z[e] = -INFINITY;
  }
}

__device__ __forceinline__ float max8(const float* z) {
  return fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7])));
}

__device__ __forceinline__ float sum8(const float* z) {
  return ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7]));
}

template <typename T, int V>
__global__ void __launch_bounds__(V == 16 ? kBiasThreads : kBiasMaxThreads, 1) bias_softmax_kernel(const __grid_constant__ BiasParams p) {
  extern __shared__ float smem[];
  float* tab = smem;                              // bias by distance, [0, near]
  float* red = smem + bias_slot(p.near) + 1;      // two words per warp
  const int gn = p.warps * 32, groups = blockDim.x / gn;
  const int group = threadIdx.x / gn, gt = threadIdx.x - group * gn;
  const int lane = threadIdx.x & 31, gw = gt >> 5;
  float* red_max = red + group * p.warps * 2;
  float* red_sum = red_max + p.warps;
  const int64_t matrix = blockIdx.x / p.ctas;
  const int cta = blockIdx.x - (int)(matrix * p.ctas);
  const float* table = p.table + (matrix % p.heads) * p.buckets;

  pdl_wait();
  for (int d = threadIdx.x; d <= p.near; d += blockDim.x) tab[bias_slot(d)] = table[bucket_of(p, d)] * kLog2e;
  __syncthreads();
  const float far = tab[bias_slot(p.near)];
  const float sl = p.scale * kLog2e;
  const int64_t base = matrix * p.rows * (int64_t)p.pitch;

  for (int i = cta * groups + group; i < p.rows; i += p.ctas * groups) {
    const int row = p.rows - 1 - i;  // the longest first
    const RowWalk w(p, row);
    const uint4* in = reinterpret_cast<const uint4*>(p.x + base + (int64_t)row * p.pitch);
    uint4* out = reinterpret_cast<uint4*>(p.out + base + (int64_t)row * p.pitch);
    const int chunks = (w.m.n + V * gn - 1) / (V * gn);
    uint4 raw[V];
    auto load = [&](int ch) {
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int j = (ch * V + q) * gn + gt;
        if (j < w.m.n) raw[q] = __ldcs(in + vector_at(w.m, j));
      }
    };
    load(0);
    zero_masked(p, w, out, gt, gn);
    float z[8];
    float m = -INFINITY;
#pragma unroll 1
    for (int ch = 0; ch < chunks; ++ch) {
      if (ch) load(ch);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int j = (ch * V + q) * gn + gt;
        if (j < w.m.n) {
          biased8<T>(p, w, tab, far, sl, vector_at(w.m, j) * 8, raw[q], z);
          m = fmaxf(m, max8(z));
        }
      }
    }
    m = redux_max(m);
    if (p.warps > 1) {
      if (lane == 0) red_max[gw] = m;
      group_sync(1 + group, gn);
      for (int k = 0; k < p.warps; ++k) m = fmaxf(m, red_max[k]);
    }
    m = fmaxf(m, -3.0e38f);  // a row of -infinity only: every exponential is 0
    float s = 0.f;
#pragma unroll 1
    for (int ch = 0; ch < chunks; ++ch) {
      if (chunks > 1) load(ch);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int j = (ch * V + q) * gn + gt;
        if (j < w.m.n) {
          biased8<T>(p, w, tab, far, sl, vector_at(w.m, j) * 8, raw[q], z);
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = ex2(z[e] - m);
          s += sum8(z);
        }
      }
    }
    s = warp_sum(s);
    if (p.warps > 1) {
      if (lane == 0) red_sum[gw] = s;
      group_sync(1 + group, gn);
      s = 0.f;
      for (int k = 0; k < p.warps; ++k) s += red_sum[k];
    }
    const float inv = s == 0.f ? 0.f : rcp_rn(s);  // a NaN stays one
#pragma unroll 1
    for (int ch = 0; ch < chunks; ++ch) {
      if (chunks > 1) load(ch);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int j = (ch * V + q) * gn + gt;
        if (j < w.m.n) {
          const int vec = vector_at(w.m, j);
          biased8<T>(p, w, tab, far, sl, vec * 8, raw[q], z);
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = ex2(z[e] - m) * inv;
          if (!((vec * 8 >= w.v.lo && vec * 8 + 8 <= w.v.hi) || vec * 8 + 8 <= w.v.s_end)) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (!sees(w.v, vec * 8 + e)) z[e] = 0.f;  // +0.0 also where the row is NaN
          }
          __stcs(out + vec, pack8<T>(z));
        }
      }
    }
  }
  pdl_trigger();
}

template <typename T, int V>
__global__ void __launch_bounds__(kBiasMaxThreads, 1) bias_backward_kernel(const __grid_constant__ BiasParams p) {
  extern __shared__ float smem[];
  const int gn = p.warps * 32, groups = blockDim.x / gn;
  const int group = threadIdx.x / gn, gt = threadIdx.x - group * gn;
  const int lane = threadIdx.x & 31, gw = gt >> 5;
  const int slots = bias_slot(p.near) + 1;
  float* acc = smem + group * slots;                      // sums by distance, [0, near)
  float* red = smem + groups * slots + group * p.warps * 2;  // two sets, used in turn
  float* far_sums = smem + groups * slots + blockDim.x / 32 * 2;  // one per warp
  const int64_t matrix = blockIdx.x / p.ctas;
  const int cta = blockIdx.x - (int)(matrix * p.ctas);
  for (int d = gt; d < slots; d += gn) acc[d] = 0.f;
  group_sync(1 + group, gn);
  pdl_wait();
  const int64_t base = matrix * p.rows * (int64_t)p.pitch;
  float far = 0.f;
  int turn = 0;

  for (int i = cta * groups + group; i < p.rows; i += p.ctas * groups) {
    const int row = p.rows - 1 - i;
    const RowWalk w(p, row);
    const uint4* in = reinterpret_cast<const uint4*>(p.x + base + (int64_t)row * p.pitch);
    const uint4* in2 = reinterpret_cast<const uint4*>(p.dp + base + (int64_t)row * p.pitch);
    uint4* out = reinterpret_cast<uint4*>(p.out + base + (int64_t)row * p.pitch);
    const int chunks = (w.m.n + V * gn - 1) / (V * gn);
    uint4 raw[V], raw2[V];
    auto load = [&](int ch) {
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int j = (ch * V + q) * gn + gt;
        if (j < w.m.n) {
          raw[q] = __ldcs(in + vector_at(w.m, j));
          raw2[q] = __ldcs(in2 + vector_at(w.m, j));
        }
      }
    };
    auto values = [&](int q, int c0, float* a, float* g) {
      unpack8<T>(raw[q], a);
      unpack8<T>(raw2[q], g);
      if (!((c0 >= w.v.lo && c0 + 8 <= w.v.hi) || c0 + 8 <= w.v.s_end)) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!sees(w.v, c0 + e)) a[e] = g[e] = 0.f;
      }
    };
    load(0);
    zero_masked(p, w, out, gt, gn);
    float a[8], g[8];
    float dot = 0.f;
#pragma unroll 1
    for (int ch = 0; ch < chunks; ++ch) {
      if (ch) load(ch);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int j = (ch * V + q) * gn + gt;
        if (j < w.m.n) {
          values(q, vector_at(w.m, j) * 8, a, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot = __fmaf_rn(a[e], g[e], dot);
        }
      }
    }
    dot = warp_sum(dot);
    if (p.warps > 1) {
      // The barrier also puts this row's additions into acc behind the last row's.
      if (lane == 0) red[turn * p.warps + gw] = dot;
      group_sync(1 + group, gn);
      dot = 0.f;
      for (int k = 0; k < p.warps; ++k) dot += red[turn * p.warps + k];
      turn ^= 1;
    }
#pragma unroll 1
    for (int ch = 0; ch < chunks; ++ch) {
      if (chunks > 1) load(ch);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const int j = (ch * V + q) * gn + gt;
        if (j < w.m.n) {
          const int vec = vector_at(w.m, j);
          values(q, vec * 8, a, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = a[e] * (g[e] - dot);
          const int d0 = w.pos - vec * 8;
          if (!((vec * 8 >= w.v.lo && vec * 8 + 8 <= w.v.hi) || vec * 8 + 8 <= w.v.s_end)) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (!sees(w.v, vec * 8 + e)) a[e] = 0.f;  // also where the row is NaN
          }
          if (d0 - 7 >= p.near) {
            far += sum8(a);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int d = d0 - e;
              if (d >= p.near) far += a[e];
              else if (d >= 0) acc[bias_slot(d)] += a[e];
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] *= p.scale;
          __stcs(out + vec, pack8<T>(a));
        }
      }
    }
    __syncwarp();  // one warp a row: this row's additions before the next row's
  }
  far = warp_sum(far);
  if (lane == 0) far_sums[threadIdx.x >> 5] = far;
  __syncthreads();
  float* partial = p.partial + (int64_t)blockIdx.x * p.buckets;
  for (int b = threadIdx.x >> 5; b < p.buckets; b += blockDim.x >> 5) {
    float s = 0.f;
    if (b == p.buckets - 1) {
      for (int k = lane; k < (int)(blockDim.x >> 5); k += 32) s += far_sums[k];
    } else {
      for (int k = 0; k < groups; ++k)
        for (int d = p.starts[b] + lane; d < p.starts[b + 1]; d += 32) s += smem[k * slots + bias_slot(d)];
    }
    s = warp_sum(s);
    if (lane == 0) partial[b] = s;
  }
  pdl_trigger();
}

struct BiasReduceParams {
  const float* partial;
  float* dtable;
  int32_t batch, heads, ctas, buckets;
};

// dtable[h, j]: one CTA per head; a warp sums a bucket's partials in 64 bits.
__global__ void __launch_bounds__(1024) bias_table_kernel(const __grid_constant__ BiasReduceParams p) {
  pdl_wait();
  const int h = blockIdx.x, lane = threadIdx.x & 31;
  const int64_t n = (int64_t)p.batch * p.ctas;
  for (int b = threadIdx.x >> 5; b < p.buckets; b += blockDim.x >> 5) {
    double s = 0.0;
    for (int64_t k = lane; k < n; k += 32) {
      const int64_t matrix = k / p.ctas * p.heads + h;
      s += (double)p.partial[(matrix * p.ctas + k % p.ctas) * p.buckets + b];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) p.dtable[h * p.buckets + b] = (float)s;
  }
}

}  // namespace cs
