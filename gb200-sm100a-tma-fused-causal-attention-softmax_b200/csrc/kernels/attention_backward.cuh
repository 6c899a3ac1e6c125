// Gradients of attention on the 5th-generation tensor core.
//
//   delta = sum over dim of d_o * o          P  = exp(scale Q K^T - lse)
//   dV = P^T d_o                             dP = d_o V^T
//   dS = P (dP - delta)                      dQ = scale dS K,  dK = scale dS^T Q
//
// Three kernels: the rows' delta; dK and dV with a tile of 128 keys per CTA
// (every sum over queries and over the heads of a group stays in one CTA's
// TMEM, or goes to memory as parts that a fourth kernel adds in order); dQ with
// a tile of 128 queries at a time. Both recompute P and dP, seven products
// instead of five, so that no sum goes through atomics: the same bits every
// time, and no fp32 copy of dQ in memory.
//
// Tiles of 128 x 128, one CTA an SM: two softmax warpgroups that take 64 columns
// of each tile, a warp of TMA loads, a warp of products. S and dP are
// fp32 in TMEM; P and dS are written over them in 16 bits and are the next
// products' first operands from there. The products are ordered so that the
// tensor core has a tile's other two while the warpgroups make P or dS. (Tiles
// of 128 x 64 with two buffers were tried first: a product of 64 columns with
// both operands in shared memory takes as long as one of 128.)
//
// 16 bits: P and dS are rounded for the tensor core. In fp16 P is taken times
// 2^15 and dS times a power of two that brings the largest possible |dS| of one sum,
// at most |d_o| |v| + |delta|, to 2^15: none overflows and small gradients keep their
// bits, also beside large ones of other sums. dQ's sums are rows, each with its own
// |d_o| and delta and the values of the key tiles that its tile sees; dK's are those of a
// tile of keys and all queries that see it. bf16 needs neither.
//
// Bound: at dim 128 a tile costs 4 x 512 tensor-core cycles in dK/dV, 3 x 512 in
// dQ, and 1024 cycles of the exponential unit in each. Measured (B200, ncu; 2 x
// 4096 queries, 16 heads over 4, window 1024, dim 128, bf16): rows 17 us, dK/dV
// 148 us at 1.65 GHz (tensor pipe active 62%), dQ 113 us at 1.66 GHz (52%).
#pragma once

#include "attention_tiles.cuh"

namespace cs {

constexpr float kHalfTop = 32768.f;  // 2^15

struct GradParams {
  CUtensorMap q, k, v, d_o;
  CUtensorMap out0, out1;    // dq; or dk, dv
  AttentionParams a;
  const float* lse2;   // [pack of heads, q_pad rows]: minus lse in units of log2; -infinity for rows without keys
  const float* delta;  // the same: minus the sum of d_o * o
  // fp16: |d_o| as lse2; [batch * heads, query_blocks], the largest |d_o| and |delta| of 64
  // queries; [batch * kv_heads, key_blocks], the largest |v| of 64 keys.
  const float* grad_norms;
  const float2* grad_tops;
  const float* value_tops;
  int32_t query_blocks, key_blocks;  // key_blocks: two a key tile
  float* partial;      // dK, dV parts of key tiles cut into several CTAs' shares
  int32_t q_pad;
  int32_t tiles;       // query (or key) tiles of a pack of heads (a kv head)
  int32_t units;       // dQ: query tiles in all
  int32_t* next;       // the next one to take; the rows kernel sets it to 0
  int32_t share;       // units of one CTA (dK, dV)
  int32_t window_shares, sink_tiles, sink_shares;  // CTAs per key tile; those of the first sink_tiles ones
};

// ---- rows: delta, lse in units of log2, norms

struct RowsParams {
  AttentionParams a;
  float* lse2;
  float* delta;
  float* grad_norms;
  float2* grad_tops;
  float* value_tops;
  int32_t* next;  // dQ's counter of query tiles
  int32_t q_pad, query_blocks, key_blocks;
};

constexpr int kRowsPerCta = 64;  // half a key tile

// The largest v of a CTA, NaN counting as nothing; words: one a warp. For thread 0.
__device__ __forceinline__ float cta_max(float v, float* words) {
  v = redux_max(v);
  __syncthreads();  // the words' last readers
  if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < 8; ++w) v = fmaxf(v, words[w]);
  return v;
}

// 16 lanes a row, four rows at a time. grid.x covers a head's tokens up to the end
// of its last tile, then (fp16) the key blocks of a kv head; grid.y = batch * heads.
template <typename T>
__global__ void __launch_bounds__(256) attention_rows_kernel(const __grid_constant__ RowsParams rp) {
  __shared__ float words[8];
  const AttentionParams& p = rp.a;
  pdl_wait();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *rp.next = 0;
  const int lane = threadIdx.x & 15, d = lane * 8;
  const bool has = d < p.head_dim;
  const int tokens = rp.q_pad >> p.pack_log2, q_ctas = (tokens + kRowsPerCta - 1) / kRowsPerCta;
  const uint4 none = make_uint4(0, 0, 0, 0);
  for (int bh = blockIdx.y; bh < p.batch * p.heads; bh += gridDim.y) {
    const int b = bh / p.heads, h = bh - b * p.heads, hk = h / p.group;
    const Lengths len(p, b);
    const int pos0 = len.position(0);
    uint4 ra[4], rg[4];
    float a[8], g[8], most = 0.f, most_delta = 0.f;
    if ((int)blockIdx.x < q_ctas) {
      const int i0 = blockIdx.x * kRowsPerCta + threadIdx.x / 16;
      const uint16_t* po = p.o.at(b, i0, h) + d;
      const uint16_t* pg = p.d_o.at(b, i0, h) + d;
      const float* plse = p.lse + (int64_t)bh * p.q_len + i0;
      const int64_t row0 = (int64_t)(bh >> p.pack_log2) * rp.q_pad + (h & ((1 << p.pack_log2) - 1));
      bool in[4];
      float lse[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + r * 16;
        in[r] = i < len.q && pos0 + i >= 0;
        ra[r] = in[r] && has ? load16(po + r * 16 * p.o.token) : none;
        rg[r] = in[r] && has ? load16(pg + r * 16 * p.d_o.token) : none;
        lse[r] = in[r] && lane == 0 ? plse[r * 16] : -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + r * 16;
        unpack8<T>(ra[r], a);
        unpack8<T>(rg[r], g);
        float dot = 0.f, norm = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dot = __fmaf_rn(a[e], g[e], dot);
          if (T::kIsHalf) norm = __fmaf_rn(g[e], g[e], norm);
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) {
          dot += __shfl_xor_sync(0xffffffffu, dot, x);
          if (T::kIsHalf) norm += __shfl_xor_sync(0xffffffffu, norm, x);
        }
        if (lane == 0 && i < tokens) {
          const int64_t row = row0 + (i << p.pack_log2);
          rp.lse2[row] = lse[r] == -INFINITY ? -INFINITY : -lse[r] * kLog2e;
          rp.delta[row] = in[r] ? -dot : 0.f;
          if (T::kIsHalf) rp.grad_norms[row] = sqrtf(norm);
        }
        if (T::kIsHalf) {
          most = fmaxf(most, norm);
          most_delta = fmaxf(most_delta, fabsf(dot));
        }
      }
      if (T::kIsHalf) {
        most = cta_max(most, words);
        most_delta = cta_max(most_delta, words);
        if (threadIdx.x == 0) rp.grad_tops[(int64_t)bh * rp.query_blocks + blockIdx.x] = make_float2(sqrtf(most), most_delta);
      }
    } else if (T::kIsHalf && h % p.group == 0) {
      const int block = (int)blockIdx.x - q_ctas, k0 = block * kRowsPerCta + threadIdx.x / 16;
      const Visible seen = sequence_keys(p, len);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int k = k0 + r * 16;
        unpack8<T>(has && sees(seen, k) ? load16(p.v.at(b, k, hk) + d) : none, a);
        float norm = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) norm = __fmaf_rn(a[e], a[e], norm);
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) norm += __shfl_xor_sync(0xffffffffu, norm, x);
        most = fmaxf(most, norm);
      }
      most = cta_max(most, words);
      if (threadIdx.x == 0) rp.value_tops[(int64_t)(b * p.kv_heads + hk) * rp.key_blocks + block] = sqrtf(most);
    }
  }
  pdl_trigger();
}

// Factor of dS in fp16: the power of two that brings a bound of |dP - delta| to at most 2^15.
__device__ __forceinline__ float ds_factor(float bound) {
  if (!(bound > 1e-30f && bound < 1e30f)) return 1.f;
  const int up = (int)((__float_as_uint(bound) >> 23) & 0xff) - 126;  // bound <= 2^up
  return __uint_as_float((uint32_t)(127 + 15 - up) << 23);
}

// P = 2^(sl s + minus_lse) of 64 columns, 0 where masked. minus_lse(e): of columns
// e and e + 1. (Packed f32x2 arithmetic: 5% off a training step against scalar.)
template <typename Lse>
__device__ __forceinline__ void scores_to_p(const uint32_t* s, bool every, uint32_t bits0, uint32_t bits1, float sl, Lse minus_lse,
                                            float* p) {
  const F2 sl2 = f2(sl, sl);
#pragma unroll
  for (int e = 0; e < 64; e += 2) {
    const float2 x = f2_out(f2_fma(f2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), sl2, minus_lse(e)));
    p[e] = ex2(x.x);
    p[e + 1] = ex2(x.y);
  }
  if (!every) {
#pragma unroll
    for (int e = 0; e < 64; ++e)
      if (!(((e < 32 ? bits0 : bits1) >> (e & 31)) & 1)) p[e] = 0.f;
  }
}

// dS = P (dP + minus_delta(e)) k1 of 32 columns in 16-bit pairs; 0 where masked,
// whatever dP holds there.
template <typename T, typename Delta>
__device__ __forceinline__ void p_to_ds(const float* p, const uint32_t* dp, bool every, uint32_t bits, float k1, Delta minus_delta,
                                        uint32_t* out) {
  const F2 k2 = f2(k1, k1);
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    F2 v = f2_add(f2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), minus_delta(e));
    if (T::kIsHalf) v = f2_mul(v, k2);
    float2 d = f2_out(f2_mul(f2(p[e], p[e + 1]), v));
    if (!every) {
      if (!((bits >> e) & 1)) d.x = 0.f;
      if (!((bits >> (e + 1)) & 1)) d.y = 0.f;
    }
    out[e / 2] = T::pack(d.x, d.y);
  }
}

constexpr int kGradThreads = 384;  // registers: 384 x 168 = 256 x 192 + 128 x 120 (dQ) = 256 x 224 + 128 x 56 (dK, dV)

// ---- dQ

struct QueryBarriers {
  uint64_t q_full, q_empty, s_full[2], dp_full, ds_full, done, dq_free, k_full[3], k_empty[3], v_full, v_empty;
  uint64_t unit_full[2], unit_empty[2];
  int32_t unit[2];    // query tiles taken; gp.units or more: no more
  uint32_t tmem, gone;
  uint32_t given_up;  // by a warpgroup's warp
};

template <int DP>
struct QuerySmem {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kKeys = 3;  // key tiles: held until dQ has used them
  static constexpr int kBytes = (2 + kKeys + 1 + 1) * kTileBytes + 256;  // Q, d_o, keys, values, the output's staging
};

// Persistent: a CTA takes the next query tile, longest first, from a counter (the
// result does not depend on who takes which); that tile's loads and first products
// run while this one's last gradients are made and brought out. The CTAs start as
// the dK/dV kernel's last ones leave, so equal shares fixed in advance would end
// unevenly: causal 4096 queries 299 us a step with them, 288 with one CTA a tile.
// Products of a tile, S in two buffers:
//   S(0) dP(0) S(1) | dQ(0) dP(1) S(2) | dQ(1) dP(2) S(3) | ...
// While the warpgroups turn S(j + 1) into P(j + 1), the tensor core has dQ(j) and
// dP(j + 1); while they make dS(j + 1), S(j + 2).
template <typename T, int DP>
__global__ void __launch_bounds__(kGradThreads, 1) attention_dq_kernel(const __grid_constant__ GradParams gp) {
  using Smem = QuerySmem<DP>;
  constexpr int kBox = kTile * 128, kTileBytes = Smem::kTileBytes, kKeys = Smem::kKeys;
  constexpr uint32_t kColumns = 512;
  extern __shared__ __align__(1024) uint8_t aligned_smem[];
  uint8_t* q_tile = aligned_smem;
  uint8_t* do_tile = q_tile + kTileBytes;
  uint8_t* k_tiles = do_tile + kTileBytes;
  uint8_t* v_tile = k_tiles + kKeys * kTileBytes;
  uint8_t* out_tile = v_tile + kTileBytes;
  QueryBarriers& bars = *reinterpret_cast<QueryBarriers*>(out_tile + kTileBytes);
  const AttentionParams& p = gp.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_addr(aligned_smem) & 1023) {  // the swizzle needs it
    if (threadIdx.x == 0) atomicOr(p.status, kStatusTimeout);
    pdl_wait();
    return;
  }
  if (warp == 8 && lane == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 1);
    mbar_init(&bars.s_full[0], 1);
    mbar_init(&bars.s_full[1], 1);
    mbar_init(&bars.dp_full, 1);
    mbar_init(&bars.ds_full, 8);
    mbar_init(&bars.done, 1);
    mbar_init(&bars.dq_free, 8);
    for (int i = 0; i < kKeys; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.unit_full[i], 1);
      mbar_init(&bars.unit_empty[i], 9);
    }
    mbar_init(&bars.v_full, 1);
    mbar_init(&bars.v_empty, 1);
    bars.gone = 0;
    bars.given_up = 0;
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
  const uint32_t tmem = bars.tmem, dp_tmem = tmem + 256, dq_tmem = tmem + 384;
  // Only the rows kernel's results are needed, and it was done before the dK/dV
  // kernel let this one start; the wait for that one is at the end.
  const Waiter wait{&bars.gone, p.status, kWaitNs};
  struct Unit {
    int bk, b, hk;
    QueryTile tile;
    Lengths len;
    TileKeys keys;
    TileList list;
    __device__ __forceinline__ Unit(const GradParams& gp, int index)
        : bk(index - gp.a.by_heads.div(index) * (int)gp.a.by_heads.by), b(gp.a.by_kv_heads.div(bk)), hk(bk - b * gp.a.kv_heads),
          tile(gp.a, hk, gp.a.by_heads.div(index), gp.tiles), len(gp.a, b), keys(gp.a, len, tile.first), list(keys) {}
  };

  // The tile of a round, for a converged warp; gp.units if the wait was given up.
  auto next_unit = [&](int round) {
    const int slot = round & 1;
    int index = gp.units;
    if (wait(&bars.unit_full[slot], (round >> 1) & 1)) index = *(volatile int32_t*)&bars.unit[slot];
    index = __shfl_sync(0xffffffffu, index, 0);
    if (lane == 0) mbar_arrive(&bars.unit_empty[slot]);
    return index;
  };

  if (warp >= 8) {
    registers_down<120>();
    if (warp == 8) {
      if (lane == 0) {
        RingPos ring;
        uint32_t tiles = 0, used = 0;  // key tiles and query tiles so far
        bool ok = true;
        for (int round = 0; ok; ++round) {
          const int slot = round & 1;
          if (!wait(&bars.unit_empty[slot], ((round >> 1) & 1) ^ 1)) break;
          const int index = atomicAdd(gp.next, 1);
          *(volatile int32_t*)&bars.unit[slot] = index;
          mbar_arrive(&bars.unit_full[slot]);
          if (index >= gp.units) break;
          const Unit u(gp, index);
          if (u.list.n == 0) continue;
          ok = wait(&bars.q_empty, (used & 1) ^ 1);
          ++used;
          if (!ok) break;
          mbar_arrive_expect_tx(&bars.q_full, 2 * kTileBytes);
#pragma unroll
          for (int box = 0; box < DP / 64; ++box) {
            tma_load(q_tile + box * kBox, &gp.q, box * 64, u.tile.head, u.tile.first, u.b, &bars.q_full);
            tma_load(do_tile + box * kBox, &gp.d_o, box * 64, u.tile.head, u.tile.first, u.b, &bars.q_full);
          }
          auto load_key = [&](int j) {
            if (!wait(&bars.k_empty[ring.s], ring.ph ^ 1)) return false;
            mbar_arrive_expect_tx(&bars.k_full[ring.s], kTileBytes);
#pragma unroll
            for (int box = 0; box < DP / 64; ++box)
              tma_load(k_tiles + ring.s * kTileBytes + box * kBox, &gp.k, box * 64, u.hk, u.list.key(j), u.b, &bars.k_full[ring.s]);
            ring.next(kKeys);
            return true;
          };
          // The order in which the products need them: K(0) V(0) K(1) | V(1) K(2) | ...
          ok = load_key(0);
          for (int j = 0; j < u.list.n && ok; ++j, ++tiles) {
            ok = wait(&bars.v_empty, (tiles & 1) ^ 1);
            if (!ok) break;
            mbar_arrive_expect_tx(&bars.v_full, kTileBytes);
#pragma unroll
            for (int box = 0; box < DP / 64; ++box)
              tma_load(v_tile + box * kBox, &gp.v, box * 64, u.hk, u.list.key(j), u.b, &bars.v_full);
            if (j + 1 < u.list.n) ok = load_key(j + 1);
          }
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      const uint32_t one = elect_one();
      auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
      RingPos ring, spent;         // key tiles: of S; of dQ
      uint32_t tiles = 0, used = 0;  // key tiles and query tiles so far
      bool ok = true;
      for (int round = 0; ok; ++round) {
        const int index = next_unit(round);
        if (index >= gp.units) break;
        const Unit u(gp, index);
        const int n = u.list.n;
        if (n == 0) continue;
        const Visible seen = sequence_keys(p, u.len);
        auto scores = [&](int j) {  // S(j)
          uint8_t* k_tile = k_tiles + ring.s * kTileBytes;
          if (!warp_wait(&bars.k_full[ring.s], ring.ph)) return false;
          clear_unseen<DP>(seen, k_tile, u.list.key(j), p.kv_len, lane);
          const uint32_t buffer = (tiles + j) & 1;
          mma_rows<T, DP, kTile>(one, tmem + buffer * 128, q_tile, kBox, k_tile, kBox);
          mma_commit(one, &bars.s_full[buffer]);
          ring.next(kKeys);
          return true;
        };
        auto products = [&](int j) {  // dP(j), the last one to read Q and d_o if j is
          if (!warp_wait(&bars.v_full, (tiles + j) & 1)) return false;
          mma_rows<T, DP, kTile>(one, dp_tmem, do_tile, kBox, v_tile, kBox);
          mma_commit(one, &bars.dp_full);
          mma_commit(one, &bars.v_empty);
          if (j == n - 1) mma_commit(one, &bars.q_empty);
          return true;
        };
        ok = warp_wait(&bars.q_full, used & 1) && scores(0) && products(0);
        if (ok && n > 1) ok = scores(1);
        if (ok && used > 0) ok = warp_wait(&bars.dq_free, (used & 1) ^ 1);  // the tile before is brought out
        tc_fence_after();
        for (int j = 0; j < n && ok; ++j) {
          ok = warp_wait(&bars.ds_full, (tiles + j) & 1);
          if (!ok) break;
          tc_fence_after();
          mma_columns<T, DP, kTile, 64>(one, dq_tmem, dp_tmem, k_tiles + spent.s * kTileBytes, kBox, j > 0);
          mma_commit(one, &bars.k_empty[spent.s]);
          spent.next(kKeys);
          if (j + 1 < n) {
            ok = products(j + 1);
            if (ok && j + 2 < n) ok = scores(j + 2);
          } else {
            mma_commit(one, &bars.done);
          }
        }
        tiles += n;
        ++used;
      }
    }
  } else {
    registers_up<192>();
    const int group = warp >> 2, in_tile = threadIdx.x & 127;  // this thread's row
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, columns = group * 64;  // and its warpgroup's columns
    const float sl = fmaxf(p.scale * kLog2e, 1.1754944e-38f);
    uint32_t tiles = 0, used = 0;
    bool ok = true;
    for (int round = 0; ok; ++round) {
      const int index = next_unit(round);
      if (index >= gp.units) break;
      const Unit u(gp, index);
      const int i = u.tile.token(in_tile);
      const Visible see = visible_keys(i < u.len.q ? u.len.position(i) : -1, u.len.kv, p.window, p.sinks);
      const int64_t row = (int64_t)((u.b * p.heads + u.tile.head) >> p.pack_log2) * gp.q_pad + (u.tile.first << p.pack_log2) + in_tile;
      // fp16: the numbers that c is made of, on their way until the first dS.
      const float* tops = gp.value_tops + (int64_t)u.bk * gp.key_blocks;
      auto top = [&](int x) { return x < 2 * u.list.n ? tops[u.list.key(x >> 1) / kRowsPerCta + (x & 1)] : 0.f; };
      float c = 1.f, values = 0.f, grad = 0.f;
      if (T::kIsHalf) {
        values = top(lane);
        grad = gp.grad_norms[row];
      }
      const F2 minus_lse = f2(gp.lse2[row], gp.lse2[row]), minus_delta = f2(gp.delta[row], gp.delta[row]);
      for (int j = 0; j < u.list.n; ++j, ++tiles) {
        const int k0 = u.list.key(j) + columns;
        const bool every = u.keys.every(u.list.key(j));
        const uint32_t bits0 = every ? 0u : visible_bits32(see, k0), bits1 = every ? 0u : visible_bits32(see, k0 + 32);
        ok = __all_sync(0xffffffffu, wait(&bars.s_full[tiles & 1], (tiles >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
        float pr[64];
        {
          uint32_t s[64];
          const uint32_t s_at = tmem + lanes + (tiles & 1) * 128 + columns;
          tmem_load32(s_at, s);
          tmem_load32(s_at + 32, s + 32);
          tmem_wait_loads();
          scores_to_p(s, every, bits0, bits1, sl, [&](int) { return minus_lse; }, pr);
        }
        if (T::kIsHalf && j == 0) {
          for (int x = lane + 32; x < 2 * u.list.n; x += 32) values = fmaxf(values, top(x));
          c = ds_factor(__fmaf_rn(grad, redux_max(values), fabsf(f2_out(minus_delta).x)));
        }
        ok = __all_sync(0xffffffffu, wait(&bars.dp_full, tiles & 1));
        if (!ok) break;
        tc_fence_after();
        const uint32_t dp_at = dp_tmem + lanes + columns;
        uint32_t dp[64], ds[32];
        tmem_load32(dp_at, dp);
        tmem_load32(dp_at + 32, dp + 32);
        tmem_wait_loads();
        p_to_ds<T>(pr, dp, every, bits0, c, [&](int) { return minus_delta; }, ds);
        p_to_ds<T>(pr + 32, dp + 32, every, bits1, c, [&](int) { return minus_delta; }, ds + 16);
        tmem_store32(dp_at, ds);  // over this warpgroup's own columns
        tmem_wait_stores();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.ds_full);
      }
      if (ok && u.list.n > 0) {
        ok = __all_sync(0xffffffffu, wait(&bars.done, used & 1));
        ++used;
      }
      // Bring the tile out, each warpgroup half of the dims. All warps go through
      // both barriers, also those that gave up waiting.
      if (threadIdx.x == 0) bulk_wait_read_all();  // the staging tile is free again
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (ok) {
        tc_fence_after();
        const bool some = u.list.n > 0 && see.hi > 0;
#pragma unroll 1
        for (int cc = group * (DP / 2); cc < (group + 1) * (DP / 2); cc += 32) {
          uint32_t o[32];
          if (u.list.n > 0) {
            tmem_load32(dq_tmem + lanes + cc, o);
            tmem_wait_loads();
          }
          stage32<T>(out_tile, in_tile, cc, o, p.scale / c, some);
        }
        tc_fence_before();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && u.list.n > 0) mbar_arrive(&bars.dq_free);
      }
      if (!ok && lane == 0) *(volatile uint32_t*)&bars.given_up = 1;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      ok = !*(volatile uint32_t*)&bars.given_up;
      if (threadIdx.x == 0 && ok) {
#pragma unroll
        for (int box = 0; box < DP / 64; ++box)
          if (box * 64 < p.head_dim) tma_store(&gp.out0, out_tile + box * kBox, box * 64, u.tile.head, u.tile.first, u.b);
        bulk_commit();
      }
    }
    if (threadIdx.x == 0) bulk_wait_all();
  }
  pdl_wait();
  finish_tmem(bars.gone, warp == 9, tmem, kColumns);
}

// ---- dK and dV

struct KeyBarriers {
  uint64_t kv_full, s_full[2], s_free, dp_full, ds_full, done, q_full[3], q_empty[3], o_full[2], o_empty[2];
  uint32_t tmem, gone;
  float factor;  // of dS, fp16
};
static_assert(sizeof(KeyBarriers) <= 256 && sizeof(QueryBarriers) <= 256, "the shared memory behind the tiles");

template <int DP>
struct KeySmem {
  static constexpr int kTileBytes = kTile * DP * 2;
  // Q is read by S, early, and by dK, late; d_o by dP and dV. With a d_o tile
  // come 128 numbers each of lse2 and delta.
  static constexpr int kQueries = 3, kGrads = 2, kGrad = kTileBytes + 1024;
  static constexpr int kBytes = (2 + kQueries) * kTileBytes + kGrads * kGrad + 256;
};

// The query tiles (units) that see a tile of keys: of one pack of heads after
// the other, `per_pack` each, from token q_first on.
struct KeyUnits {
  int32_t q_first, per_pack, n, step;  // step: tokens of a query tile
  int32_t every_lo, every_hi;          // tokens [every_lo, every_hi) see all 128 keys
  __device__ __forceinline__ KeyUnits(const AttentionParams& p, const Lengths& len, int k0) {
    step = kTile >> p.pack_log2;
    q_first = per_pack = n = every_lo = every_hi = 0;
    if (k0 >= len.kv || len.q <= 0) return;
    const int64_t pos0 = len.position(0), k1 = min(k0 + kTile, len.kv) - 1;
    const int64_t lo = max((int64_t)0, k0 - pos0);
    int64_t hi = len.q, all = len.q;
    if (p.window) {
      if (k0 >= p.sinks) hi = min(hi, k1 + p.window - pos0);
      if (k0 + kTile > p.sinks) all = min(all, max((int64_t)k0, (int64_t)p.sinks) + p.window - pos0);
    }
    if (lo >= hi) return;
    q_first = (int)lo / step * step;
    per_pack = ((int)hi + step - 1) / step - (int)lo / step;
    n = per_pack * (p.group >> p.pack_log2);
    every_lo = (int)max((int64_t)0, k0 + kTile - 1 - pos0);
    every_hi = k0 + kTile <= len.kv ? (int)max(all, (int64_t)0) : 0;
  }
};

// Columns of a query tile, first token i0, that token t is at or behind.
__device__ __forceinline__ int column_of(int t, int i0, int pack_log2) { return min(max(t - i0, 0), kTile) << pack_log2; }

// Queries [lo, hi) of a sequence see key k.
__device__ __forceinline__ void queries_of(const AttentionParams& p, const Lengths& len, int k, int& lo, int& hi) {
  const int64_t pos0 = len.position(0);
  lo = (int)min(max((int64_t)0, k - pos0), (int64_t)len.q);
  hi = len.q;
  if (p.window && k >= p.sinks) hi = (int)min((int64_t)hi, max((int64_t)0, (int64_t)k + p.window - pos0));
  if (k >= len.kv) hi = lo;
}

// S(u), then dP(u), then P(u) and dS(u) live in the half (u & 1) of 256 columns,
// each written once the warpgroups have read the one before. Products in this
// order:
//   S(0) S(1) dP(0) | dV(0) dP(1) dK(0) S(2) | dV(1) dP(2) dK(1) S(3) | ...
// While the warpgroups turn S(u + 1) into P(u + 1) (kept in registers) the tensor
// core has dV(u), dP(u + 1) and dK(u); while they make dS(u + 1), S(u + 2).
// Measured in cycles a tile: P over S, so that S(u + 1) waits for dV(u), 3400; P
// and dS over dP, so that dP(u + 1) waits for dK(u), 3290; this one 2950, most of them
// the warpgroups' (P 1300, dS 1200), the tensor core's four products 2160.
template <typename T, int DP>
__global__ void __launch_bounds__(kGradThreads, 1) attention_dkv_kernel(const __grid_constant__ GradParams gp) {
  using Smem = KeySmem<DP>;
  constexpr int kBox = kTile * 128, kTileBytes = Smem::kTileBytes, kQueries = Smem::kQueries, kGrads = Smem::kGrads, kGrad = Smem::kGrad;
  constexpr uint32_t kColumns = 512;
  constexpr float kShift = T::kIsHalf ? 15.f : 0.f;
  extern __shared__ __align__(1024) uint8_t aligned_smem[];
  uint8_t* k_tile = aligned_smem;
  uint8_t* v_tile = k_tile + kTileBytes;
  uint8_t* q_tiles = v_tile + kTileBytes;
  uint8_t* grads = q_tiles + kQueries * kTileBytes;
  KeyBarriers& bars = *reinterpret_cast<KeyBarriers*>(grads + kGrads * kGrad);
  const AttentionParams& p = gp.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_addr(aligned_smem) & 1023) {
    if (threadIdx.x == 0) atomicOr(p.status, kStatusTimeout);
    return;
  }
  if (warp == 8 && lane == 0) {
    mbar_init(&bars.kv_full, 1);
    mbar_init(&bars.s_full[0], 1);
    mbar_init(&bars.s_full[1], 1);
    mbar_init(&bars.s_free, 8);
    mbar_init(&bars.dp_full, 1);
    mbar_init(&bars.ds_full, 8);
    mbar_init(&bars.done, 1);
    for (int i = 0; i < kQueries; ++i) {
      mbar_init(&bars.q_full[i], 1);
      mbar_init(&bars.q_empty[i], 1);
    }
    for (int i = 0; i < kGrads; ++i) {
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.o_empty[i], 1);
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
  const int bk = blockIdx.x % (p.batch * p.kv_heads), which = blockIdx.x / (p.batch * p.kv_heads);
  const int b = bk / p.kv_heads, hk = bk - b * p.kv_heads;
  const int in_sinks = gp.sink_tiles * gp.sink_shares;
  const int tile = which < in_sinks ? which / gp.sink_shares : gp.sink_tiles + (which - in_sinks) / gp.window_shares;
  const int share = which < in_sinks ? which % gp.sink_shares : (which - in_sinks) % gp.window_shares;
  const int k0 = tile * kTile;
  const Lengths len(p, b);
  const KeyUnits units(p, len, k0);
  const int u0 = min(share * gp.share, units.n), n = min(units.n - u0, gp.share);
  const Waiter wait{&bars.gone, p.status, kWaitNs};

  if (n > 0 || share == 0) {
    if (warp >= 8) {
      registers_down<56>();
      if (warp == 8) {
        if (lane == 0 && n > 0) {
          mbar_arrive_expect_tx(&bars.kv_full, 2 * kTileBytes);
#pragma unroll
          for (int box = 0; box < DP / 64; ++box) {
            tma_load(k_tile + box * kBox, &gp.k, box * 64, hk, k0, b, &bars.kv_full);
            tma_load(v_tile + box * kBox, &gp.v, box * 64, hk, k0, b, &bars.kv_full);
          }
          RingPos q_at, o_at;
          auto load_query = [&](int u) {
            const int pack = u / units.per_pack, i0 = units.q_first + (u - pack * units.per_pack) * units.step;
            const int head = hk * p.group + (pack << p.pack_log2);
            if (!wait(&bars.q_empty[q_at.s], q_at.ph ^ 1)) return false;
            mbar_arrive_expect_tx(&bars.q_full[q_at.s], kTileBytes);
#pragma unroll
            for (int box = 0; box < DP / 64; ++box)
              tma_load(q_tiles + q_at.s * kTileBytes + box * kBox, &gp.q, box * 64, head, i0, b, &bars.q_full[q_at.s]);
            q_at.next(kQueries);
            return true;
          };
          auto load_grad = [&](int u) {
            const int pack = u / units.per_pack, i0 = units.q_first + (u - pack * units.per_pack) * units.step;
            const int head = hk * p.group + (pack << p.pack_log2);
            if (!wait(&bars.o_empty[o_at.s], o_at.ph ^ 1)) return false;
            uint8_t* to = grads + o_at.s * kGrad;
            mbar_arrive_expect_tx(&bars.o_full[o_at.s], kGrad);
#pragma unroll
            for (int box = 0; box < DP / 64; ++box)
              tma_load(to + box * kBox, &gp.d_o, box * 64, head, i0, b, &bars.o_full[o_at.s]);
            const int64_t row = (int64_t)((b * p.heads + head) >> p.pack_log2) * gp.q_pad + (i0 << p.pack_log2);
            bulk_g2s(to + kTileBytes, gp.lse2 + row, 512, &bars.o_full[o_at.s]);
            bulk_g2s(to + kTileBytes + 512, gp.delta + row, 512, &bars.o_full[o_at.s]);
            o_at.next(kGrads);
            return true;
          };
          // In the order in which the products need them.
          bool ok = load_query(u0);
          for (int u = u0; u < u0 + n && ok; ++u) {
            ok = load_grad(u);
            if (ok && u + 1 < u0 + n) ok = load_query(u + 1);
          }
        }
        __syncwarp();
      } else if (warp == 9 && n > 0) {
        const uint32_t one = elect_one();
        auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
        const int q_lo = max(0, -len.position(0));  // queries before it are at negative positions
        RingPos q_next, q_used, o_next, o_used;  // of S and of dK; of dP and of dV
        int q_sub = u0 % units.per_pack, o_sub = q_sub;
        // Zero the rows of a tile that are no queries of the sequence.
        auto clean = [&](uint8_t* tile, int& sub) {
          const int i0 = units.q_first + sub * units.step;
          if (++sub == units.per_pack) sub = 0;
          const int first = column_of(q_lo, i0, p.pack_log2), end = column_of(len.q, i0, p.pack_log2);
          if (first > 0 || (end < kTile && len.q < p.q_len))  // (the copy wrote zeros behind q_len)
            clear_rows<DP>(tile, lane, [&](int r) { return r >= first && r < end; });
        };
        auto scores = [&](int u) {  // S(u)
          uint8_t* q_tile = q_tiles + q_next.s * kTileBytes;
          if (!warp_wait(&bars.q_full[q_next.s], q_next.ph)) return false;
          clean(q_tile, q_sub);
          mma_rows<T, DP, kTile>(one, tmem + (u & 1) * 128, k_tile, kBox, q_tile, kBox);
          mma_commit(one, &bars.s_full[u & 1]);
          q_next.next(kQueries);
          return true;
        };
        auto products = [&](int u) {  // dP(u)
          uint8_t* o_tile = grads + o_next.s * kGrad;
          if (!warp_wait(&bars.o_full[o_next.s], o_next.ph)) return false;
          clean(o_tile, o_sub);
          if (!warp_wait(&bars.s_free, u & 1)) return false;
          tc_fence_after();
          mma_rows<T, DP, kTile>(one, tmem + (u & 1) * 128, v_tile, kBox, o_tile, kBox);
          mma_commit(one, &bars.dp_full);
          o_next.next(kGrads);
          return true;
        };
        bool ok = warp_wait(&bars.kv_full, 0) && scores(0);
        if (ok && n > 1) ok = scores(1);
        if (ok) ok = products(0);
        for (int u = 0; u < n && ok; ++u) {
          const uint32_t at = tmem + (u & 1) * 128;
          if (!warp_wait(&bars.ds_full, u & 1)) break;
          tc_fence_after();
          // Each stage is given back as soon as its last product is in the queue:
          // loads take most of a tile's time.
          mma_columns<T, DP, kTile, 64>(one, dv_tmem, at, grads + o_used.s * kGrad, kBox, u > 0);
          mma_commit(one, &bars.o_empty[o_used.s]);
          if (u + 1 < n && !products(u + 1)) break;
          mma_columns<T, DP, kTile, 64>(one, dk_tmem, at + 32, q_tiles + q_used.s * kTileBytes, kBox, u > 0);
          mma_commit(one, u + 1 < n ? &bars.q_empty[q_used.s] : &bars.done);
          if (u + 2 < n) ok = scores(u + 2);
          o_used.next(kGrads);
          q_used.next(kQueries);
        }
      } else if (T::kIsHalf && warp == 10 && n > 0) {
        // The factor of dS, from all queries that see the tile.
        const float* norms = gp.value_tops + (int64_t)bk * gp.key_blocks + tile * 2;
        const float v = fmaxf(norms[0], norms[1]);
        const int first = units.q_first / kRowsPerCta;
        const int blocks = (units.q_first + units.per_pack * units.step - 1) / kRowsPerCta - first + 1;
        const float2* tops = gp.grad_tops + (int64_t)(b * p.heads + hk * p.group) * gp.query_blocks + first;
        float most = 0.f;
#pragma unroll 4
        for (int x = lane; x < blocks * p.group; x += 32) {
          const int h = x / blocks;
          const float2 top = tops[(int64_t)h * gp.query_blocks + (x - h * blocks)];
          most = fmaxf(most, __fmaf_rn(top.x, v, top.y));
        }
        most = redux_max(most);
        if (lane == 0) bars.factor = ds_factor(most);
        asm volatile("bar.arrive 3, 288;" ::: "memory");
      }
    } else {
      registers_up<224>();
      const int group = warp >> 2, row = threadIdx.x & 127;  // this thread's key
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const int columns = group * 64;  // this warpgroup's queries of a tile
      const float sl = fmaxf(p.scale * kLog2e, 1.1754944e-38f);
      float c = 1.f;
      if (T::kIsHalf && n > 0) {
        asm volatile("bar.sync 3, 288;" ::: "memory");
        c = bars.factor;
      }
      const float k1 = T::kIsHalf ? c * (1.f / kHalfTop) : 1.f;
      int q_lo, q_hi;
      queries_of(p, len, k0 + row, q_lo, q_hi);
      bool ok = true;
      static_assert(kGrads == 2, "a unit's d_o stage is u & 1");
      const int i_end = units.q_first + units.per_pack * units.step;
      int i0 = n > 0 ? units.q_first + u0 % units.per_pack * units.step : 0;
      for (int u = 0; u < n; ++u, i0 = i0 + units.step == i_end ? units.q_first : i0 + units.step) {
        const float* rows = reinterpret_cast<const float*>(grads + (u & 1) * kGrad + kTileBytes) + columns;
        const bool every = i0 >= units.every_lo && i0 + units.step <= units.every_hi;
        const int c_lo = column_of(q_lo, i0, p.pack_log2) - columns, c_hi = column_of(q_hi, i0, p.pack_log2) - columns;
        uint32_t bits0 = 0, bits1 = 0;
        if (!every) {
          bits0 = below_bits(c_hi) & ~below_bits(c_lo);
          bits1 = below_bits(c_hi - 32) & ~below_bits(c_lo - 32);
        }
        float4 quad;
        auto pair = [&](int e) {  // two queries' numbers, read four at a time
          if (!(e & 2)) quad = *reinterpret_cast<const float4*>(rows + e);
          return e & 2 ? f2(quad.z, quad.w) : f2(quad.x, quad.y);
        };
        ok = __all_sync(0xffffffffu, wait(&bars.o_full[u & 1], (u >> 1) & 1) && wait(&bars.s_full[u & 1], (u >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
        const uint32_t at = tmem + lanes + (u & 1) * 128 + columns;
        float pr[64];
        {
          uint32_t s[64];
          tmem_load32(at, s);
          tmem_load32(at + 32, s + 32);
          tmem_wait_loads();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.s_free);
          scores_to_p(s, every, bits0, bits1, sl, [&](int e) { return T::kIsHalf ? f2_add(pair(e), f2(kShift, kShift)) : pair(e); }, pr);
        }
        ok = __all_sync(0xffffffffu, wait(&bars.dp_full, u & 1));
        if (!ok) break;
        tc_fence_after();
        // P goes over the first half of this warpgroup's dP columns, dS over the second.
        uint32_t dp[32], ds[16], out[16];
        tmem_load32(at, dp);
        tmem_wait_loads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int e = 0; e < 16; ++e) out[e] = T::pack(pr[h * 32 + 2 * e], pr[h * 32 + 2 * e + 1]);
          tmem_store16(at + h * 16, out);
        }
        p_to_ds<T>(pr, dp, every, bits0, k1, [&](int e) { return pair(128 + e); }, ds);
        tmem_load32(at + 32, dp);
        tmem_wait_loads();
        tmem_store16(at + 32, ds);
        p_to_ds<T>(pr + 32, dp, every, bits1, k1, [&](int e) { return pair(160 + e); }, out);
        tmem_store16(at + 48, out);
        tmem_wait_stores();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.ds_full);
      }
      if (ok && n > 0) ok = __all_sync(0xffffffffu, wait(&bars.done, 0));
      if (ok) {
        // Warpgroup 0 brings out dV, warpgroup 1 dK.
        tc_fence_after();
        const uint32_t from = (group ? dk_tmem : dv_tmem) + lanes;
        const float factor = group ? p.scale / c : T::kIsHalf ? 1.f / kHalfTop : 1.f;
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
            stage32<T>(group ? k_tile : v_tile, row, cc, o, factor, n > 0 && q_lo < q_hi);
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
#pragma unroll 8
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
