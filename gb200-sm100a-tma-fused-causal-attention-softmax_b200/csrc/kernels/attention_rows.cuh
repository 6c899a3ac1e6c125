// Gradients of attention, one warp per row: the plain form of the formulas.
//
// Lane l holds dims 4 l .. 4 l + 3 of a row; a score is a warp sum.
#pragma once

#include "attention.cuh"

namespace cs {

template <typename T>
__device__ __forceinline__ float4 load_dims(const uint16_t* row, int lane, int dim) {
  if (lane * 4 >= dim) return make_float4(0.f, 0.f, 0.f, 0.f);
  const uint2 r = *reinterpret_cast<const uint2*>(row + lane * 4);
  const float2 a = T::unpack(r.x), b = T::unpack(r.y);
  return make_float4(a.x, a.y, b.x, b.y);
}

template <typename T>
__device__ __forceinline__ void store_dims(uint16_t* row, int lane, int dim, float4 f) {
  if (lane * 4 < dim) *reinterpret_cast<uint2*>(row + lane * 4) = make_uint2(T::pack(f.x, f.y), T::pack(f.z, f.w));
}

__device__ __forceinline__ float dot4(float4 a, float4 b) {
  return warp_sum(__fmaf_rn(a.x, b.x, __fmaf_rn(a.y, b.y, __fmaf_rn(a.z, b.z, a.w * b.w))));
}

__device__ __forceinline__ void add4(float4& a, float s, float4 b) {
  a.x = __fmaf_rn(s, b.x, a.x);
  a.y = __fmaf_rn(s, b.y, a.y);
  a.z = __fmaf_rn(s, b.z, a.z);
  a.w = __fmaf_rn(s, b.w, a.w);
}

__device__ __forceinline__ float4 times4(float4 a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }

// dq and delta, one warp per query; grid.y = batch * heads.
template <typename T>
__global__ void __launch_bounds__(128) attention_dq_rows_kernel(const __grid_constant__ AttentionParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31, i = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i >= p.q_len) return;
  for (int bh = blockIdx.y; bh < p.batch * p.heads; bh += gridDim.y) {
    const int b = bh / p.heads, h = bh - b * p.heads, hk = h / p.group;
    const Lengths n(p, b);
    const Visible v = visible_keys(i < n.q ? n.position(i) : -1, n.kv, p.window, p.sinks);
    const float4 q = load_dims<T>(p.q.at(b, i, h), lane, p.head_dim);
    const float4 g = load_dims<T>(p.d_o.at(b, i, h), lane, p.head_dim);
    const float delta = dot4(g, load_dims<T>(p.o.at(b, i, h), lane, p.head_dim));
    const float lse = p.lse[(int64_t)bh * p.q_len + i] * kLog2e;
    const float sl = p.scale * kLog2e;
    float4 dq = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = v.s_end > 0 ? 0 : v.lo; k < v.hi; ++k) {
      if (k == v.s_end && (k = v.lo) >= v.hi) break;
      const float4 key = load_dims<T>(p.k.at(b, k, hk), lane, p.head_dim);
      const float e = ex2(__fmaf_rn(dot4(q, key), sl, -lse));
      const float dp = dot4(g, load_dims<T>(p.v.at(b, k, hk), lane, p.head_dim));
      add4(dq, e * (dp - delta), key);
    }
    store_dims<T>(p.dq.at(b, i, h), lane, p.head_dim, times4(dq, p.scale));
    if (lane == 0) p.delta[(int64_t)bh * p.q_len + i] = delta;
  }
}

// dk and dv, one warp per key.
template <typename T>
__global__ void __launch_bounds__(128) attention_dkv_rows_kernel(const __grid_constant__ AttentionParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31, k = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (k >= p.kv_len) return;
  for (int bh = blockIdx.y; bh < p.batch * p.kv_heads; bh += gridDim.y) {
    const int b = bh / p.kv_heads, hk = bh - b * p.kv_heads;
    const Lengths n(p, b);
    float4 dk = make_float4(0.f, 0.f, 0.f, 0.f), dv = dk;
    if (k < n.kv) {
      const float4 key = load_dims<T>(p.k.at(b, k, hk), lane, p.head_dim);
      const float4 val = load_dims<T>(p.v.at(b, k, hk), lane, p.head_dim);
      const float sl = p.scale * kLog2e;
      for (int h = hk * p.group; h < (hk + 1) * p.group; ++h)
        for (int i = max(0, k - n.position(0)); i < n.q; ++i) {
          if (!sees(visible_keys(n.position(i), n.kv, p.window, p.sinks), k)) {
            if (p.window && k >= p.sinks) break;  // no later query sees it either
            continue;
          }
          const int64_t row = ((int64_t)b * p.heads + h) * p.q_len + i;
          const float4 q = load_dims<T>(p.q.at(b, i, h), lane, p.head_dim);
          const float4 g = load_dims<T>(p.d_o.at(b, i, h), lane, p.head_dim);
          const float e = ex2(__fmaf_rn(dot4(q, key), sl, -p.lse[row] * kLog2e));
          add4(dv, e, g);
          add4(dk, e * (dot4(g, val) - p.delta[row]), q);
        }
    }
    store_dims<T>(p.dk.at(b, k, hk), lane, p.head_dim, times4(dk, p.scale));
    store_dims<T>(p.dv.at(b, k, hk), lane, p.head_dim, dv);
  }
}

}  // namespace cs
