// Gradients of attention on the 5th-generation tensor core.
//
//   delta = sum over dim of d_o * o          P  = exp(scale Q K^T - lse)
//   dV = P^T d_o                             dP = d_o V^T
//   dS = P (dP - delta)                      dQ = scale dS K,  dK = scale dS^T Q
//
// Three kernels: the rows' delta; dK and dV with a tile of 128 keys per CTA
// (every sum over queries and over the heads of a group stays in one CTA's
// TMEM); dQ with a tile of 128 queries per CTA. Both recompute P and dP, seven
// products instead of five, so that no sum crosses CTAs: no atomics, the same
// bits every time, and no fp32 copy of dQ in memory.
//
// The streamed operand comes in tiles of 64 rows: S and dP of 128 x 64, P and
// dS written over them in 16 bits as the next products' first operands (TMEM).
//
// 16 bits: P and dS are rounded for the tensor core. In fp16 P is taken times
// 2^15 and dS times a power of two, from the largest norms of d_o and v rows of
// the kv head, that brings the largest possible |dS| to 2^15: small gradients
// keep their bits and none overflows. bf16 needs neither.
//
// Bound: at dim 128 a 128 x 64 tile costs 4 x 256 tensor-core cycles in dK/dV
// and 3 x 256 in dQ; the two S-like products (64 columns, both operands in
// shared memory) are held back by shared memory, 384 cycles each.
#pragma once

#include "attention_tiles.cuh"

namespace cs {

constexpr int kSub = 64;             // rows of a streamed tile
constexpr float kHalfTop = 32768.f;  // 2^15

struct GradParams {
  CUtensorMap q, k, v, d_o;  // stationary: 128 rows; streamed: 64
  CUtensorMap out0, out1;    // dq; or dk, dv
  AttentionParams a;
  const float* lse2;   // [batch * heads, q_pad]: minus lse in units of log2; -infinity for rows without keys
  const float* delta;  // the same: minus the sum of d_o * o
  const float* norms;  // fp16: [2, batch * kv_heads], largest |d_o| and |v| of a row
  float* partial;      // dK, dV parts of key tiles cut into several CTAs' shares
  int32_t q_pad;
  int32_t tiles;       // query (or key) tiles
  int32_t share;       // units of one CTA (dK, dV)
  int32_t window_shares, sink_tiles, sink_shares;  // CTAs per key tile; those of the first sink_tiles ones
};

// ---- rows: delta, lse in units of log2, norms

struct RowsParams {
  AttentionParams a;
  float* lse2;
  float* delta;
  uint32_t* norms;  // as integers: the bits of non-negative floats order like them
  int32_t q_pad;
};

__device__ __forceinline__ void raise_max(uint32_t* at, float v) {
  const float m = redux_max(v);  // NaN counts as nothing
  if ((threadIdx.x & 31) == 0 && m > 0.f) atomicMax(at, __float_as_uint(m));
}

// 16 lanes a row. grid.x covers q_pad rows of a head, then (fp16) the rows of a
// kv head; grid.y = batch * heads.
template <typename T>
__global__ void __launch_bounds__(256) attention_rows_kernel(const __grid_constant__ RowsParams rp) {
  const AttentionParams& p = rp.a;
  pdl_wait();
  const int lane = threadIdx.x & 15, d = lane * 8, per_cta = 16;
  const int q_ctas = (rp.q_pad + per_cta - 1) / per_cta;
  for (int bh = blockIdx.y; bh < p.batch * p.heads; bh += gridDim.y) {
    const int b = bh / p.heads, h = bh - b * p.heads, hk = h / p.group;
    const Lengths len(p, b);
    float a[8], g[8];
    if ((int)blockIdx.x < q_ctas) {
      const int i = blockIdx.x * per_cta + threadIdx.x / 16;
      const bool in = i < len.q && len.position(i) >= 0;
      float dot = 0.f, norm = 0.f;
      if (in && d < p.head_dim) {
        unpack8<T>(*reinterpret_cast<const uint4*>(p.o.at(b, i, h) + d), a);
        unpack8<T>(*reinterpret_cast<const uint4*>(p.d_o.at(b, i, h) + d), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dot = __fmaf_rn(a[e], g[e], dot);
          norm = __fmaf_rn(g[e], g[e], norm);
        }
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) {
        dot += __shfl_xor_sync(0xffffffffu, dot, x);
        norm += __shfl_xor_sync(0xffffffffu, norm, x);
      }
      if (lane == 0 && i < rp.q_pad) {
        const float lse = in ? p.lse[(int64_t)bh * p.q_len + i] : -INFINITY;
        rp.lse2[(int64_t)bh * rp.q_pad + i] = lse == -INFINITY ? -INFINITY : -lse * kLog2e;
        rp.delta[(int64_t)bh * rp.q_pad + i] = in ? -dot : 0.f;
      }
      if (T::kIsHalf) raise_max(rp.norms + b * p.kv_heads + hk, norm);
    } else if (T::kIsHalf && h % p.group == 0) {
      const int k = (blockIdx.x - q_ctas) * per_cta + threadIdx.x / 16;
      float norm = 0.f;
      if (k < len.kv && d < p.head_dim && sees(sequence_keys(p, len), k)) {
        unpack8<T>(*reinterpret_cast<const uint4*>(p.v.at(b, k, hk) + d), a);
#pragma unroll
        for (int e = 0; e < 8; ++e) norm = __fmaf_rn(a[e], a[e], norm);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) norm += __shfl_xor_sync(0xffffffffu, norm, x);
      raise_max(rp.norms + p.batch * p.kv_heads + b * p.kv_heads + hk, norm);
    }
  }
  pdl_trigger();
}

// Factor of dS: 1, or in fp16 the power of two that brings the bound
// |dP - delta| <= 2 |d_o| |v| to at most 2^15.
template <typename T>
__device__ __forceinline__ float ds_factor(const GradParams& g, int bk) {
  if (!T::kIsHalf) return 1.f;
  const float top = 2.f * sqrtf(g.norms[bk]) * sqrtf(g.norms[g.a.batch * g.a.kv_heads + bk]);
  if (!(top > 1e-30f && top < 1e30f)) return 1.f;
  const int up = (int)((__float_as_uint(top) >> 23) & 0xff) - 126;  // top <= 2^up
  return __uint_as_float((uint32_t)(127 + 15 - up) << 23);
}

// P and dS of 32 columns: scores s and dp in, packed pairs out.
// minus_lse: shift - lse2 of columns e and e + 1; minus_delta: - delta.
// P = 2^(sl s + minus_lse), dS = P (dp + minus_delta) k1.
template <typename T, typename Lse, typename Delta>
__device__ __forceinline__ void grad32(const uint32_t* s, const uint32_t* dp, bool every, uint32_t bits, float sl, float k1,
                                       Lse minus_lse, Delta minus_delta, uint32_t* p_out, uint32_t* ds_out) {
  const F2 sl2 = f2(sl, sl), k2 = f2(k1, k1);
  float p[32], d[32];
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const float2 x = f2_out(f2_fma(f2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), sl2, minus_lse(e)));
    p[e] = ex2(x.x);
    p[e + 1] = ex2(x.y);
    F2 v = f2_add(f2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), minus_delta(e));
    if (T::kIsHalf) v = f2_mul(v, k2);
    const float2 y = f2_out(f2_mul(f2(p[e], p[e + 1]), v));
    d[e] = y.x;
    d[e + 1] = y.y;
  }
  if (!every) {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (!((bits >> e) & 1)) p[e] = d[e] = 0.f;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    p_out[e] = T::pack(p[2 * e], p[2 * e + 1]);
    ds_out[e] = T::pack(d[2 * e], d[2 * e + 1]);
  }
}

// Stage 32 columns of this thread's row (128-byte swizzle, box of 128 rows).
template <typename T>
__device__ __forceinline__ void stage32(uint8_t* tile, int row, int c, const uint32_t* v, float factor, bool some) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t w[4];
#pragma unroll
    for (int h = 0; h < 4; ++h)
      w[h] = some ? T::pack(__uint_as_float(v[8 * e + 2 * h]) * factor, __uint_as_float(v[8 * e + 2 * h + 1]) * factor) : 0u;
    const int chunk = (c & 63) / 8 + e;
    *reinterpret_cast<uint4*>(tile + (c >> 6) * (kTile * 128) + row * 128 + ((chunk ^ (row & 7)) << 4)) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- dQ: like the forward kernel, two CTAs an SM

struct QueryBarriers {
  uint64_t q_full, s_full, ds_full, dq_full, k_full[2], k_empty[2], v_full, v_empty;
  uint32_t tmem, gone;
};

template <int DP>
struct QuerySmem {
  static constexpr int kFixed = kTile * DP * 2, kSubBytes = kSub * DP * 2;
  // Exactly what two CTAs an SM allow at dim 128: the base is 1024-aligned by itself.
  static constexpr int kBytes = 2 * kFixed + 3 * kSubBytes + 256;
};

template <typename T, int DP>
__global__ void __launch_bounds__(256, 2) attention_dq_kernel(const __grid_constant__ GradParams gp) {
  constexpr int kBox = kTile * 128, kSubBox = kSub * 128, kFixed = QuerySmem<DP>::kFixed, kSubBytes = QuerySmem<DP>::kSubBytes;
  constexpr uint32_t kColumns = 256;
  extern __shared__ __align__(1024) uint8_t aligned_smem[];
  uint8_t* q_tile = aligned_smem;
  uint8_t* do_tile = q_tile + kFixed;
  uint8_t* k_tiles = do_tile + kFixed;
  uint8_t* v_tile = k_tiles + 2 * kSubBytes;
  QueryBarriers& bars = *reinterpret_cast<QueryBarriers*>(v_tile + kSubBytes);
  const AttentionParams& p = gp.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_addr(aligned_smem) & 1023) {  // the swizzle needs it
    if (threadIdx.x == 0) atomicOr(p.status, kStatusTimeout);
    return;
  }
  if (warp == 4 && lane == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.s_full, 1);
    mbar_init(&bars.ds_full, 4);
    mbar_init(&bars.dq_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
    }
    mbar_init(&bars.v_full, 1);
    mbar_init(&bars.v_empty, 1);
    bars.gone = 0;
    fence_barrier_init();
    prefetch_map(&gp.q);
    prefetch_map(&gp.d_o);
    prefetch_map(&gp.k);
    prefetch_map(&gp.v);
  }
  if (warp == 5) tmem_alloc(&bars.tmem, kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem, s_tmem = tmem, dp_tmem = tmem + 64, dq_tmem = tmem + 128;
  // Only the rows kernel's results are needed, and it was done before the dK/dV
  // kernel let this one start; the wait for that one is at the end.

  const int bk = blockIdx.x % (p.batch * p.kv_heads), unit = blockIdx.x / (p.batch * p.kv_heads);
  const int b = bk / p.kv_heads, hk = bk - b * p.kv_heads;
  const int head = hk * p.group + unit % p.group, first = (gp.tiles - 1 - unit / p.group) * kTile;
  const Lengths len(p, b);
  const TileKeys keys(p, len, first);
  const TileList<kSub> list(keys);
  const Waiter wait{&bars.gone, p.status, kWaitNs};

  if (warp >= 4) {
    registers_down<96>();
    if (warp == 4) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars.q_full, 2 * kFixed);
#pragma unroll
        for (int box = 0; box < DP / 64; ++box) {
          tma_load(q_tile + box * kBox, &gp.q, box * 64, head, first, b, &bars.q_full);
          tma_load(do_tile + box * kBox, &gp.d_o, box * 64, head, first, b, &bars.q_full);
        }
        RingPos ring;
        for (int j = 0; j < list.n; ++j, ring.next(2)) {
          const int k0 = list.key(j);
          if (!wait(&bars.k_empty[ring.s], ring.ph ^ 1)) break;
          mbar_arrive_expect_tx(&bars.k_full[ring.s], kSubBytes);
#pragma unroll
          for (int box = 0; box < DP / 64; ++box)
            tma_load(k_tiles + ring.s * kSubBytes + box * kSubBox, &gp.k, box * 64, hk, k0, b, &bars.k_full[ring.s]);
          if (!wait(&bars.v_empty, (j & 1) ^ 1)) break;
          mbar_arrive_expect_tx(&bars.v_full, kSubBytes);
#pragma unroll
          for (int box = 0; box < DP / 64; ++box)
            tma_load(v_tile + box * kSubBox, &gp.v, box * 64, hk, k0, b, &bars.v_full);
        }
      }
      __syncwarp();
    } else if (warp == 5) {
      const Visible seen = sequence_keys(p, len);
      const uint32_t one = elect_one();
      auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
      bool ok = warp_wait(&bars.q_full, 0);
      RingPos ring;
      for (int j = 0; j <= list.n && ok; ++j) {
        uint8_t* k_tile = k_tiles + ring.s * kSubBytes;
        uint8_t* k_last = k_tiles + (ring.s ^ 1) * kSubBytes;
        if (j < list.n) {
          if (!warp_wait(&bars.k_full[ring.s], ring.ph)) break;
          clear_unseen<DP, kSub>(seen, k_tile, list.key(j), lane);
          if (!warp_wait(&bars.v_full, j & 1)) break;
        }
        if (j > 0) {
          if (!warp_wait(&bars.ds_full, (j - 1) & 1)) break;
          tc_fence_after();
          mma_columns<T, DP, kSub, 16>(one, dq_tmem, dp_tmem, k_last, kSubBox, j > 1);
        }
        if (j < list.n) {
          mma_rows<T, DP, kSub>(one, s_tmem, q_tile, kBox, k_tile, kSubBox);
          mma_rows<T, DP, kSub>(one, dp_tmem, do_tile, kBox, v_tile, kSubBox);
          mma_commit(one, &bars.s_full);
          mma_commit(one, &bars.v_empty);
          if (j > 0) mma_commit(one, &bars.k_empty[ring.s ^ 1]);
        } else {
          mma_commit(one, &bars.dq_full);
        }
        ring.next(2);
      }
    }
  } else {
    registers_up<160>();
    const int i = first + threadIdx.x;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const Visible see = visible_keys(i < len.q ? len.position(i) : -1, len.kv, p.window, p.sinks);
    const float sl = fmaxf(p.scale * kLog2e, 1.1754944e-38f);
    const int64_t row = ((int64_t)b * p.heads + head) * gp.q_pad + i;
    const float c = ds_factor<T>(gp, bk);
    const float lse = i < gp.q_pad ? gp.lse2[row] : -INFINITY, delta = i < gp.q_pad ? gp.delta[row] : 0.f;
    const F2 minus_lse = f2(lse, lse), minus_delta = f2(delta, delta);
    bool ok = true;
    for (int j = 0; j < list.n; ++j) {
      const int k0 = list.key(j);
      ok = __all_sync(0xffffffffu, wait(&bars.s_full, j & 1));
      if (!ok) break;
      tc_fence_after();
      const bool every = keys.template every<kSub>(k0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t s[32], dp[32], pp[16], ds[16];
        tmem_load32(s_tmem + lanes + h * 32, s);
        tmem_load32(dp_tmem + lanes + h * 32, dp);
        tmem_wait_loads();
        grad32<T>(s, dp, every, every ? 0u : visible_bits32(see, k0 + h * 32), sl, c, [&](int) { return minus_lse; }, [&](int) { return minus_delta; }, pp, ds);
        tmem_store16(dp_tmem + lanes + h * 16, ds);
      }
      tmem_wait_stores();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.ds_full);
    }
    if (ok) ok = __all_sync(0xffffffffu, wait(&bars.dq_full, 0));
    if (ok) {
      tc_fence_after();
      const bool some = list.n > 0 && see.hi > 0;
#pragma unroll 1
      for (int cc = 0; cc < DP; cc += 32) {
        uint32_t o[32];
        if (list.n > 0) {
          tmem_load32(dq_tmem + lanes + cc, o);
          tmem_wait_loads();
        }
        stage32<T>(q_tile, threadIdx.x, cc, o, p.scale / c, some);
      }
      fence_proxy_async_smem();
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (threadIdx.x == 0 && !*(volatile uint32_t*)&bars.gone) {
#pragma unroll
      for (int box = 0; box < DP / 64; ++box)
        if (box * 64 < p.head_dim) tma_store(&gp.out0, q_tile + box * kBox, box * 64, head, first, b);
      bulk_commit();
      bulk_wait_all();
    }
  }
  pdl_wait();
  finish_tmem(bars.gone, warp == 5, tmem, kColumns);
}

// ---- dK and dV: one CTA an SM. Two warpgroups take half of the columns each, so
// that P and dS are there by the time the tensor core is through with the last
// unit's gradients and the next one's scores (two buffers); taking the units in
// turn instead left it waiting a third of the time.

struct KeyBarriers {
  uint64_t kv_full, s_full[2], ds_full[2], done, q_full[4], q_empty[4];
  uint32_t tmem, gone;
};

template <int DP>
struct KeySmem {
  static constexpr int kFixed = kTile * DP * 2, kSubBytes = kSub * DP * 2;
  static constexpr int kStage = 2 * kSubBytes + 1024;  // Q, d_o, 64 lse2, 64 delta
  static constexpr int kStages = 4;
  static constexpr int kBytes = 2 * kFixed + kStages * kStage + 256;
};

// The (head, 64 queries) units that see a tile of keys, heads first.
struct KeyUnits {
  int32_t q_first, per_head, n;  // q_first: of a head's first unit
  int32_t every_lo, every_hi;    // queries [every_lo, every_hi) see all 128 keys
  __device__ __forceinline__ KeyUnits(const AttentionParams& p, const Lengths& len, int k0) {
    q_first = per_head = n = every_lo = every_hi = 0;
    if (k0 >= len.kv || len.q <= 0) return;
    const int64_t pos0 = len.position(0), k1 = min(k0 + kTile, len.kv) - 1;
    const int64_t lo = max((int64_t)0, k0 - pos0);
    int64_t hi = len.q, all = len.q;
    if (p.window) {
      if (k0 >= p.sinks) hi = min(hi, k1 + p.window - pos0);
      if (k0 + kTile > p.sinks) all = min(all, max((int64_t)k0, (int64_t)p.sinks) + p.window - pos0);
    }
    if (lo >= hi) return;
    q_first = (int)(lo / kSub) * kSub;
    per_head = (int)((hi + kSub - 1) / kSub - lo / kSub);
    n = per_head * p.group;
    every_lo = (int)max((int64_t)0, k0 + kTile - 1 - pos0);
    every_hi = k0 + kTile <= len.kv ? (int)max(all, (int64_t)0) : 0;
  }
};

// Queries [lo, hi) of a sequence see key k.
__device__ __forceinline__ void queries_of(const AttentionParams& p, const Lengths& len, int k, int& lo, int& hi) {
  const int64_t pos0 = len.position(0);
  lo = (int)min(max((int64_t)0, k - pos0), (int64_t)len.q);
  hi = len.q;
  if (p.window && k >= p.sinks) hi = (int)min((int64_t)hi, max((int64_t)0, (int64_t)k + p.window - pos0));
  if (k >= len.kv) hi = lo;
}

template <typename T, int DP>
__global__ void __launch_bounds__(384, 1) attention_dkv_kernel(const __grid_constant__ GradParams gp) {
  using Smem = KeySmem<DP>;
  constexpr int kBox = kTile * 128, kSubBox = kSub * 128, kFixed = Smem::kFixed, kSubBytes = Smem::kSubBytes, kStages = Smem::kStages;
  constexpr uint32_t kColumns = 512;
  constexpr float kShift = T::kIsHalf ? 15.f : 0.f;
  extern __shared__ __align__(1024) uint8_t aligned_smem[];
  uint8_t* k_tile = aligned_smem;
  uint8_t* v_tile = k_tile + kFixed;
  uint8_t* stages = v_tile + kFixed;
  KeyBarriers& bars = *reinterpret_cast<KeyBarriers*>(stages + kStages * Smem::kStage);
  const AttentionParams& p = gp.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_addr(aligned_smem) & 1023) {
    if (threadIdx.x == 0) atomicOr(p.status, kStatusTimeout);
    return;
  }
  if (warp == 8 && lane == 0) {
    mbar_init(&bars.kv_full, 1);
    mbar_init(&bars.done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.ds_full[i], 8);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.q_full[i], 1);
      mbar_init(&bars.q_empty[i], 1);
    }
    bars.gone = 0;
    fence_barrier_init();
    prefetch_map(&gp.q);
    prefetch_map(&gp.d_o);
    prefetch_map(&gp.k);
    prefetch_map(&gp.v);
  }
  if (warp == 9) tmem_alloc(&bars.tmem, kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem, dv_tmem = tmem + 256, dk_tmem = dv_tmem + DP;
  pdl_wait();
  pdl_trigger();  // dQ's CTAs may take the SMs that this kernel's last ones leave

  // Which key tile and which share of its units; a kv head's CTAs are apart, so
  // that neighbours in time read the same queries.
  const int bk = blockIdx.x % (p.batch * p.kv_heads), at = blockIdx.x / (p.batch * p.kv_heads);
  const int b = bk / p.kv_heads, hk = bk - b * p.kv_heads;
  const int in_sinks = gp.sink_tiles * gp.sink_shares;
  const int tile = at < in_sinks ? at / gp.sink_shares : gp.sink_tiles + (at - in_sinks) / gp.window_shares;
  const int share = at < in_sinks ? at % gp.sink_shares : (at - in_sinks) % gp.window_shares;
  const int k0 = tile * kTile;
  const Lengths len(p, b);
  const KeyUnits units(p, len, k0);
  const int u0 = min(share * gp.share, units.n), n = min(units.n - u0, gp.share);
  const Waiter wait{&bars.gone, p.status, kWaitNs};

  if (n > 0 || share == 0) {
  if (warp >= 8) {
    registers_down<152>();
    if (warp == 8) {
      if (lane == 0 && n > 0) {
        mbar_arrive_expect_tx(&bars.kv_full, 2 * kFixed);
#pragma unroll
        for (int box = 0; box < DP / 64; ++box) {
          tma_load(k_tile + box * kBox, &gp.k, box * 64, hk, k0, b, &bars.kv_full);
          tma_load(v_tile + box * kBox, &gp.v, box * 64, hk, k0, b, &bars.kv_full);
        }
        RingPos ring;
        for (int u = u0; u < u0 + n; ++u, ring.next(kStages)) {
          const int h = u / units.per_head, i0 = units.q_first + (u - h * units.per_head) * kSub, head = hk * p.group + h;
          uint8_t* stage = stages + ring.s * Smem::kStage;
          if (!wait(&bars.q_empty[ring.s], ring.ph ^ 1)) break;
          mbar_arrive_expect_tx(&bars.q_full[ring.s], 2 * kSubBytes + 512);
#pragma unroll
          for (int box = 0; box < DP / 64; ++box) {
            tma_load(stage + box * kSubBox, &gp.q, box * 64, head, i0, b, &bars.q_full[ring.s]);
            tma_load(stage + kSubBytes + box * kSubBox, &gp.d_o, box * 64, head, i0, b, &bars.q_full[ring.s]);
          }
          const int64_t row = ((int64_t)b * p.heads + head) * gp.q_pad + i0;
          bulk_g2s(stage + 2 * kSubBytes, gp.lse2 + row, 256, &bars.q_full[ring.s]);
          bulk_g2s(stage + 2 * kSubBytes + 256, gp.delta + row, 256, &bars.q_full[ring.s]);
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      const uint32_t one = elect_one();
      auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
      const int q_lo = max(0, -len.position(0));  // queries before it are at negative positions
      bool ok = n > 0 && warp_wait(&bars.kv_full, 0);
      RingPos next, ring;  // of the scores; of the gradients, one unit behind
      int sub = n > 0 ? u0 % units.per_head : 0;
      for (int u = 0; u <= n && ok; ++u) {
        if (u < n) {
          uint8_t* stage = stages + next.s * Smem::kStage;
          if (!warp_wait(&bars.q_full[next.s], next.ph)) break;
          const int i0 = units.q_first + sub * kSub;
          if (++sub == units.per_head) sub = 0;
          if (i0 < q_lo || i0 + kSub > len.q) {
            auto keep = [&](int r) { return i0 + r >= q_lo && i0 + r < len.q; };
            clear_rows<DP, kSub>(stage, lane, keep);
            clear_rows<DP, kSub>(stage + kSubBytes, lane, keep);
          }
          // The buffer is free: unit u - 2's gradients are ahead in the queue.
          const uint32_t s = tmem + (u & 1) * 128;
          mma_rows<T, DP, kSub>(one, s, k_tile, kBox, stage, kSubBox);
          mma_rows<T, DP, kSub>(one, s + 64, v_tile, kBox, stage + kSubBytes, kSubBox);
          mma_commit(one, &bars.s_full[u & 1]);
          next.next(kStages);
        }
        if (u > 0) {
          const int w = u - 1;
          uint8_t* stage = stages + ring.s * Smem::kStage;
          if (!warp_wait(&bars.ds_full[w & 1], (w >> 1) & 1)) break;
          tc_fence_after();
          const uint32_t s = tmem + (w & 1) * 128;
          mma_columns<T, DP, kSub, 32>(one, dv_tmem, s, stage + kSubBytes, kSubBox, w > 0);
          mma_columns<T, DP, kSub, 32>(one, dk_tmem, s + 64, stage, kSubBox, w > 0);
          mma_commit(one, w == n - 1 ? &bars.done : &bars.q_empty[ring.s]);
          ring.next(kStages);
        }
      }
    }
  } else {
    registers_up<176>();
    const int group = warp >> 2, row = threadIdx.x & 127;  // warpgroup; this thread's key
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t half = tmem + lanes + group * 32;  // this warpgroup's columns of the first buffer's S
    const float sl = fmaxf(p.scale * kLog2e, 1.1754944e-38f);
    const float c = ds_factor<T>(gp, bk), k1 = T::kIsHalf ? c * (1.f / kHalfTop) : 1.f;
    int q_lo, q_hi;
    queries_of(p, len, k0 + row, q_lo, q_hi);
    bool ok = true;
    int sub = n > 0 ? u0 % units.per_head : 0;
    RingPos ring;
    for (int u = 0; u < n; ++u, ring.next(kStages)) {
      const int i0 = units.q_first + sub * kSub;
      if (++sub == units.per_head) sub = 0;
      const float* rows = reinterpret_cast<const float*>(stages + ring.s * Smem::kStage + 2 * kSubBytes) + group * 32;
      ok = __all_sync(0xffffffffu, wait(&bars.q_full[ring.s], ring.ph) && wait(&bars.s_full[u & 1], (u >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      const bool every = i0 >= units.every_lo && i0 + kSub <= units.every_hi;
      const uint32_t s_at = half + (u & 1) * 128, dp_at = s_at + 64;
      uint32_t s[32], dp[32], pp[16], ds[16];
      tmem_load32(s_at, s);
      tmem_load32(dp_at, dp);
      const int at = i0 + group * 32;
      const uint32_t bits = every ? 0u : below_bits(q_hi - at) & ~below_bits(q_lo - at);
      tmem_wait_loads();
      const F2 shift2 = f2(kShift, kShift);
      auto pair = [&](int e) {  // two rows' numbers
        const float2 v = *reinterpret_cast<const float2*>(rows + e);
        return f2(v.x, v.y);
      };
      grad32<T>(s, dp, every, bits, sl, k1, [&](int e) { return T::kIsHalf ? f2_add(pair(e), shift2) : pair(e); },
                [&](int e) { return pair(64 + e); }, pp, ds);
      tmem_store16(s_at, pp);  // over this warpgroup's own columns
      tmem_store16(dp_at, ds);
      tmem_wait_stores();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.ds_full[u & 1]);
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, wait(&bars.done, 0));
    if (ok) {
      // Warpgroup 0 brings out dV, warpgroup 1 dK.
      tc_fence_after();
      const uint32_t from = (group ? dk_tmem : dv_tmem) + lanes;
      const float factor = group ? p.scale / c : T::kIsHalf ? 1.f / kHalfTop : 1.f;
      uint8_t* tile_smem = group ? k_tile : v_tile;
      const bool whole = units.n <= gp.share;
      float4* part = reinterpret_cast<float4*>(gp.partial) + ((int64_t)blockIdx.x * 2 + group) * (kTile * DP / 4) + row;
#pragma unroll 1
      for (int cc = 0; cc < DP; cc += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_load32(from + cc, o);
          tmem_wait_loads();
        }
        if (whole) {
          stage32<T>(tile_smem, row, cc, o, factor, n > 0 && q_lo < q_hi);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            part[(cc / 4 + e) * kTile] =
                make_float4(__uint_as_float(o[4 * e]) * factor, __uint_as_float(o[4 * e + 1]) * factor,
                            __uint_as_float(o[4 * e + 2]) * factor, __uint_as_float(o[4 * e + 3]) * factor);
        }
      }
      fence_proxy_async_smem();
    }
    asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
    if (row == 0 && units.n <= gp.share && !*(volatile uint32_t*)&bars.gone) {
#pragma unroll
      for (int box = 0; box < DP / 64; ++box)
        if (box * 64 < p.head_dim)
          tma_store(group ? &gp.out0 : &gp.out1, (group ? k_tile : v_tile) + box * kBox, box * 64, hk, k0, b);
      bulk_commit();
      bulk_wait_all();
    }
  }
  }
  finish_tmem(bars.gone, warp == 9, tmem, kColumns);
}

// Sum of a cut key tile's parts, in order. grid.x: as the first share of every
// key tile that may be cut; threads: 4 columns of a key each.
template <typename T, int DP>
__global__ void __launch_bounds__(256) attention_dkv_join_kernel(const __grid_constant__ GradParams gp) {
  const AttentionParams& p = gp.a;
  const int heads = p.batch * p.kv_heads;
  const int bk = blockIdx.x % heads, tile = blockIdx.x / heads, b = bk / p.kv_heads, hk = bk - b * p.kv_heads;
  pdl_wait();
  const Lengths len(p, b);
  const KeyUnits units(p, len, tile * kTile);
  if (units.n <= gp.share) return;
  const int shares = (units.n + gp.share - 1) / gp.share;
  const int first = tile < gp.sink_tiles ? tile * gp.sink_shares
                                         : gp.sink_tiles * gp.sink_shares + (tile - gp.sink_tiles) * gp.window_shares;
  for (int x = blockIdx.y * blockDim.x + threadIdx.x; x < 2 * kTile * DP / 4; x += gridDim.y * blockDim.x) {
    const int which = x / (kTile * DP / 4), at = x - which * (kTile * DP / 4), d = at / kTile * 4, row = at % kTile;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < shares; ++s) {
      const int64_t cta = (int64_t)(first + s) * heads + bk;
      const float4 v = reinterpret_cast<const float4*>(gp.partial)[(cta * 2 + which) * (kTile * DP / 4) + at];
      sum.x += v.x;
      sum.y += v.y;
      sum.z += v.z;
      sum.w += v.w;
    }
    const int k = tile * kTile + row;
    int lo, hi;
    queries_of(p, len, k, lo, hi);
    if (k < p.kv_len && d < p.head_dim)
      *reinterpret_cast<uint2*>((which ? p.dk : p.dv).at(b, k, hk) + d) =
          lo < hi ? make_uint2(T::pack(sum.x, sum.y), T::pack(sum.z, sum.w)) : make_uint2(0, 0);
  }
}

}  // namespace cs
