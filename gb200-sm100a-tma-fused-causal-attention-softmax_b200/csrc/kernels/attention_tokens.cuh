// Attention of few queries over many keys: single tokens reading a cache.
//
// The query rows that share a kv head, (query, head) pairs, are at most 8 NT;
// a CTA reads a share ("split") of their visible keys and its warps take 16 keys in turn, each with its own running maximum, sum and
// output; warps are joined in shared memory, splits by a second kernel.
// Bound: HBM, each visible key and value read once.
//
// Products run on mma m16n8k16 with keys (then dims) as the 16 rows and the
// query rows as the 8 columns: 8 rows fill it, so one token of a group of up to
// 8 heads wastes little, and a tcgen05 tile of 128 rows would be empty but for
// a sixteenth. Fragments come straight from global memory in 16-byte loads:
// the order of dims within a sum is free, so a lane takes 8 consecutive dims
// of a key as two steps' worth, and the same dims of a query row. Values are
// read 8 dims of four keys a lane, and pairs of keys are put together by byte
// permutes. Nothing is staged in shared memory; 12 warps an SM with a step's
// keys and values in flight (4 to 8 KB each) cover the latency.
//
// The running maximum of a column moves only when a score passes it by more
// than 2^8, so most steps need no reduction across lanes. For the second product
// probabilities are two 16-bit numbers, the rounded one and the rest, so that they
// keep 16 (bf16) or 22 bits and the output's own rounding is the only one to speak of
// (fp16: times 2^7, so that small ones keep their bits: 2^8 2^7 < 65504); sums and
// outputs are fp32. Measured without / with the rest: error 2.3e-3 / 1.7e-3 of the
// output in bf16, 2.8e-4 / 2.1e-4 in fp16; 64 tokens of 32 heads over 8, window 4096,
// 163.8 / 165.4 us; 32 of 16 heads over 2048 keys, dim 64, 48.0 / 49.5; 4 x 2 over
// 16384, 32 heads over 4, 32.8 / 34.7.
#pragma once

#include "attention.cuh"

namespace cs {

constexpr int kTokenWarps = 4;
constexpr float kMaxLag = 8.f;  // in units of log2

struct TokenParams {
  AttentionParams a;
  float* part_o;      // [kv head, split, 8 NT, DP]
  float* part_stats;  // [kv head, split, 8 NT, 2]: maximum (log2 units), sum
  int32_t splits;
  int32_t rows;       // 8 NT
  int32_t dim_pad;    // DP
};

template <typename T>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (T::kIsHalf)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 block of 16-bit elements held two a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The steps of 16 keys that hold the visible keys, numbered densely.
struct KeySteps {
  Visible u;  // union over the rows
  int32_t n_sink, w_beg, n;
  __device__ __forceinline__ KeySteps(const AttentionParams& p, const Lengths& len) {
    u.s_end = u.lo = u.hi = 0;
    if (len.q > 0) {
      const Visible first = visible_keys(len.position(0), len.kv, p.window, p.sinks);
      u = visible_keys(len.position(len.q - 1), len.kv, p.window, p.sinks);
      u.lo = min(u.lo, first.lo);
      u.s_end = min(u.s_end, u.lo);
    }
    const int s = (u.s_end + 15) >> 4;
    w_beg = u.lo < u.hi ? u.lo >> 4 : s;
    n_sink = min(s, w_beg);
    n = n_sink + (u.lo < u.hi ? ((u.hi + 15) >> 4) - w_beg : s - n_sink);
  }
  __device__ __forceinline__ int key(int j) const { return (j < n_sink ? j : j - n_sink + w_beg) * 16; }
};

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(kTokenWarps * 32, NT == 1 ? 3 : 2) attention_tokens_kernel(const __grid_constant__ TokenParams tp) {
  constexpr int KC = DP / 32, VC = DP / 64, MT = DP / 16, kRows = 8 * NT;
  constexpr float kShift = T::kIsHalf ? 7.f : 0.f;
  __shared__ __align__(16) float sm_o[kTokenWarps][kRows][DP + 4];
  __shared__ float sm_m[kTokenWarps][kRows], sm_l[kTokenWarps][kRows];
  const AttentionParams& p = tp.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int bk = blockIdx.x / tp.splits, split = blockIdx.x - bk * tp.splits;
  const int b = bk / p.kv_heads, hk = bk - b * p.kv_heads;
  const int rows = p.q_len * p.group;
  pdl_wait();
  const Lengths len(p, b);
  const KeySteps steps(p, len);
  const int begin = (int)((int64_t)steps.n * split / tp.splits), end = (int)((int64_t)steps.n * (split + 1) / tp.splits);
  const float sl = p.scale * kLog2e;

  // This lane's query row of each column tile (as B), and the masks of the two
  // columns whose scores it holds.
  uint4 q[NT][KC];
  Visible see[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = n * 8 + g, i = r / p.group;
    const uint16_t* src = p.q.at(b, i, hk * p.group + r - i * p.group);
#pragma unroll
    for (int c = 0; c < KC; ++c)
      q[n][c] = r < rows && i < len.q && c * 32 + t * 8 < p.head_dim ? load16(src + c * 32 + t * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = n * 8 + 2 * t + e, ci = col / p.group;
      see[n][e] = visible_keys(col < rows && ci < len.q ? len.position(ci) : -1, len.kv, p.window, p.sinks);
    }
  }

  float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
  }

  const uint16_t* kbase = p.k.at(b, 0, hk) + t * 8;
  const uint16_t* vbase = p.v.at(b, 0, hk) + g * 8;
  const bool full = p.head_dim == DP;
  uint4 kf[2][KC];
  auto load_keys = [&](int key0) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int key = key0 + g + 8 * e;
      const bool in = sees(steps.u, key);
      const uint16_t* src = kbase + (int64_t)key * p.k.token;
#pragma unroll
      for (int c = 0; c < KC; ++c)
        kf[e][c] = in && (full || c * 32 + t * 8 < p.head_dim) ? load16(src + c * 32) : make_uint4(0, 0, 0, 0);
    }
  };
  if (begin + warp < end) load_keys(steps.key(begin + warp));
  for (int j = begin + warp; j < end; j += kTokenWarps) {
    const int key0 = steps.key(j);
    uint4 vf[4][VC];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int key = key0 + 2 * t + (e & 1) + 8 * (e >> 1);
      const bool in = sees(steps.u, key);
      const uint16_t* src = vbase + (int64_t)key * p.v.token;
#pragma unroll
      for (int c = 0; c < VC; ++c)
        vf[e][c] = in && (full || c * 64 + g * 8 < p.head_dim) ? load16(src + c * 64) : make_uint4(0, 0, 0, 0);
    }
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        mma16816<T>(s[n], kf[0][c].x, kf[1][c].x, kf[0][c].y, kf[1][c].y, q[n][c].x, q[n][c].y);
        mma16816<T>(s[n], kf[0][c].z, kf[1][c].z, kf[0][c].w, kf[1][c].w, q[n][c].z, q[n][c].w);
      }
    }
    if (j + kTokenWarps < end) load_keys(steps.key(j + kTokenWarps));
    bool above = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // keys g (e < 2) and g + 8, columns 2 t and 2 t + 1
        s[n][e] = sees(see[n][e & 1], key0 + g + (e >> 1) * 8) ? s[n][e] * sl : -INFINITY;
        above |= s[n][e] > m[n][e & 1] + kMaxLag;
      }
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          top = fmaxf(top, m[n][e]);
          f[e] = top == -INFINITY ? 1.f : ex2(m[n][e] - top);
          m[n][e] = top;
          l[n][e] *= f[e];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][i][e] *= f[e & 1];
      }
    }
    uint32_t pb[NT][2], rest[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float at = m[n][e & 1] == -INFINITY ? 0.f : m[n][e & 1];  // nothing seen yet: -infinity stays
        s[n][e] = ex2(s[n][e] - at + kShift);
        l[n][e & 1] += s[n][e];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t most = T::pack(s[n][2 * e], s[n][2 * e + 1]);
        const float2 f = T::unpack(most);
        pb[n][e] = transpose8(most);
        rest[n][e] = transpose8(T::pack(s[n][2 * e] - f.x, s[n][2 * e + 1] - f.y));
      }
    }
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      const uint32_t w[4][4] = {{vf[0][c].x, vf[0][c].y, vf[0][c].z, vf[0][c].w},
                                {vf[1][c].x, vf[1][c].y, vf[1][c].z, vf[1][c].w},
                                {vf[2][c].x, vf[2][c].y, vf[2][c].z, vf[2][c].w},
                                {vf[3][c].x, vf[3][c].y, vf[3][c].z, vf[3][c].w}};
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // rows g and g + 8 of tile 4 c + i: dims 64 c + 8 g + 2 i and + 1
        const uint32_t a0 = __byte_perm(w[0][i], w[1][i], 0x5410), a1 = __byte_perm(w[0][i], w[1][i], 0x7632);
        const uint32_t a2 = __byte_perm(w[2][i], w[3][i], 0x5410), a3 = __byte_perm(w[2][i], w[3][i], 0x7632);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816<T>(o[n][4 * c + i], a0, a1, a2, a3, pb[n][0], pb[n][1]);
          mma16816<T>(o[n][4 * c + i], a0, a1, a2, a3, rest[n][0], rest[n][1]);
        }
      }
    }
  }

  // Join the warps.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
      const int r = n * 8 + 2 * t + e;
      if (g == 0) {
        sm_m[warp][r] = m[n][e];
        sm_l[warp][r] = l[n][e];
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int d = (i >> 2) * 64 + g * 8 + (i & 3) * 2;
        *reinterpret_cast<float2*>(&sm_o[warp][r][d]) = make_float2(o[n][i][e], o[n][i][e + 2]);
      }
    }
  __syncthreads();
  constexpr int kLanes = DP / 4;  // 4 dims a thread
  for (int r = threadIdx.x / kLanes; r < rows; r += kTokenWarps * 32 / kLanes) {
    const int d = (threadIdx.x % kLanes) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kTokenWarps; ++w) top = fmaxf(top, sm_m[w][r]);
    float sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kTokenWarps; ++w) {
      const float f = sm_m[w][r] == -INFINITY ? 0.f : ex2(sm_m[w][r] - top);
      const float4 x = *reinterpret_cast<const float4*>(&sm_o[w][r][d]);
      sum = __fmaf_rn(f, sm_l[w][r], sum);
      v.x = __fmaf_rn(f, x.x, v.x);
      v.y = __fmaf_rn(f, x.y, v.y);
      v.z = __fmaf_rn(f, x.z, v.z);
      v.w = __fmaf_rn(f, x.w, v.w);
    }
    if (tp.splits > 1) {
      const int64_t at = (int64_t)blockIdx.x * kRows + r;
      *reinterpret_cast<float4*>(tp.part_o + at * DP + d) = v;
      // -infinity: no key seen; a NaN among the scores goes on in the sum.
      if (d == 0) *reinterpret_cast<float2*>(tp.part_stats + at * 2) = make_float2(top == -INFINITY && sum != 0.f ? 0.f : top, sum);
    } else {
      const int i = r / p.group, h = hk * p.group + r - i * p.group;
      const float inv = sum == 0.f ? 0.f : rcp_rn(sum);
      if (sum == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);  // 0 times another row's NaN among the values
      if (d < p.head_dim)
        *reinterpret_cast<uint2*>(p.o.at(b, i, h) + d) = make_uint2(T::pack(v.x * inv, v.y * inv), T::pack(v.z * inv, v.w * inv));
      if (d == 0 && p.lse)
        p.lse[((int64_t)b * p.heads + h) * p.q_len + i] = sum == 0.f ? -INFINITY : (top - kShift + __log2f(sum)) * (1.f / kLog2e);
    }
  }
  pdl_trigger();
}

// Joins the splits: one CTA per row. Weights first, then the warps take splits in
// turn, lanes hold 4 dims each: all loads are independent.
constexpr int kMaxSplits = 2048;

template <typename T, int kWarps>
__global__ void __launch_bounds__(kWarps * 32) attention_join_kernel(const __grid_constant__ TokenParams tp) {
  constexpr float kShift = T::kIsHalf ? 7.f : 0.f;
  constexpr int kJoinThreads = kWarps * 32;
  __shared__ __align__(16) float sm_v[kWarps][128 + 4];
  __shared__ float weight[kMaxSplits], words[kWarps];
  const AttentionParams& p = tp.a;
  const int rows = p.q_len * p.group, bk = blockIdx.x / rows, row = blockIdx.x - bk * rows;
  const int b = bk / p.kv_heads, hk = bk - b * p.kv_heads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = lane * 4;
  const int64_t first = (int64_t)bk * tp.splits * tp.rows + row;  // of the splits' rows
  pdl_wait();
  // The maximum, the weights, the sum.
  float top = -INFINITY;
  for (int s = threadIdx.x; s < tp.splits; s += kJoinThreads) {
    weight[s] = tp.part_stats[(first + (int64_t)s * tp.rows) * 2];
    top = fmaxf(top, weight[s]);
  }
  top = redux_max(top);
  if (lane == 0) words[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, words[w]);
  __syncthreads();
  float sum = 0.f;
  for (int s = threadIdx.x; s < tp.splits; s += kJoinThreads) {
    const bool none = weight[s] == -INFINITY;
    const float f = none ? 0.f : ex2(weight[s] - top);
    weight[s] = f;
    if (!none) sum = __fmaf_rn(f, tp.part_stats[(first + (int64_t)s * tp.rows) * 2 + 1], sum);  // a NaN goes on at any weight
  }
  sum = warp_sum(sum);
  if (lane == 0) words[warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += words[w];
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d < tp.dim_pad) {
#pragma unroll 8
    for (int s = warp; s < tp.splits; s += kWarps) {
      const float4 x = *reinterpret_cast<const float4*>(tp.part_o + (first + (int64_t)s * tp.rows) * tp.dim_pad + d);
      const float f = weight[s];
      if (f != 0.f) {  // a split without keys may hold anything
        v.x = __fmaf_rn(f, x.x, v.x);
        v.y = __fmaf_rn(f, x.y, v.y);
        v.z = __fmaf_rn(f, x.z, v.z);
        v.w = __fmaf_rn(f, x.w, v.w);
      }
    }
  }
  *reinterpret_cast<float4*>(&sm_v[warp][d]) = v;
  __syncthreads();
  const int i = row / p.group, h = hk * p.group + row - i * p.group;
  const float inv = sum == 0.f ? 0.f : rcp_rn(sum);
  if (threadIdx.x < p.head_dim / 2) {
    float2 o = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      o.x += sm_v[w][threadIdx.x * 2];
      o.y += sm_v[w][threadIdx.x * 2 + 1];
    }
    *reinterpret_cast<uint32_t*>(p.o.at(b, i, h) + threadIdx.x * 2) = T::pack(o.x * inv, o.y * inv);
  }
  if (threadIdx.x == 0 && p.lse)
    p.lse[((int64_t)b * p.heads + h) * p.q_len + i] = sum == 0.f ? -INFINITY : (top - kShift + __log2f(sum)) * (1.f / kLog2e);
}

}  // namespace cs
