// Attention of many queries: tiles of 128 queries x 128 keys on the
// 5th-generation tensor core.
//
// A tile's 128 rows are (token, head) pairs: 128 / pack tokens of `pack` heads
// that read the same keys, the largest power of two in the group. Few tokens
// fill a tile that way, and the keys of a window that only some rows see are
// fewer. A CTA owns one such tile and streams key and value tiles through a ring
// of shared-memory stages; two CTAs share an SM. Where tiles are few and their
// keys many, several CTAs share a tile's keys and a second kernel joins them.
//
//   warps 0-3: softmax, one thread per query; they hold a row of 128 scores
//   warp 4:    TMA loads     warp 5: products (one thread)     6, 7: no work
//
// The second four give registers to the first: 128 x 176 + 128 x 80 = 256 x 128.
//
// Per key tile: S = Q K^T (TMEM, fp32) -> the softmax warps read their rows and
// write P over S as 16-bit pairs -> O += P V with P from TMEM. S of the next key
// tile follows P V in the tensor core's queue, so S overwrites P only after its
// use, and once S is there O is complete and may be rescaled. While one CTA is
// in its softmax the tensor core works for the other, whose start and end it
// also covers. Measured against one CTA an SM with two query tiles that share
// each key tile (half the L2 traffic): 16384 queries x 16 heads, window 4096,
// dim 128: 468 us against 509; dim 64: 425 against 459; 512 over 8192: 112
// against 147. Both sides then issued products under a branch on the lane, which cost
// the one warp with two tiles' products more; with a converged warp (451 us for the
// first case in a short replay) the second form has not been measured. (A query in
// two threads, 64 keys of a tile each: 440, 374 and 104 against 435, 362 and 105 of
// one thread. At dim 128 the power limit holds the clock down: 1.62 GHz in a second
// of these calls, 1.95 at dim 64.)
//
// Running maximum: it moves only when a row passes it by more than 2^8, so the
// output in TMEM is rescaled rarely (all sums are relative to the same
// maximum, so the result does not depend on it). P is rounded to 16 bits for
// the tensor core, fp16 after a factor of 2^7 that keeps small probabilities
// out of its subnormals; sums are fp32 over unrounded values.
//
// Bound: at dim 128 a tile pair costs 1024 tensor-core cycles (two products of
// 2 128^3 at 8192 a cycle) and 1024 cycles of the exponential unit (128^2 at
// 16 a cycle), at dim 64 512 and 1024.
#pragma once

#include "attention.cuh"
#include "tcgen05.cuh"

namespace cs {

constexpr int kTile = 128;

struct TileParams {
  CUtensorMap q, k, v, o;
  AttentionParams a;
  int32_t q_tiles;      // per pack of heads
  int32_t splits;       // CTAs per query tile
  float* part_o;        // splits > 1: [CTA, DP / 4, 128 rows, 4]
  float* part_stats;    // [CTA, 128 rows, 2]: maximum (log2 units), sum
};

// A tile of queries: its first token and head.
struct QueryTile {
  int32_t first, head, pack_log2;
  __device__ __forceinline__ QueryTile(const AttentionParams& p, int hk, int unit, int tiles) {
    pack_log2 = p.pack_log2;
    const int tile = p.by_packs.div(unit);
    first = (tiles - 1 - tile) * (kTile >> pack_log2);  // the latest first: they see most
    head = hk * p.group + ((unit - tile * (int)p.by_packs.by) << pack_log2);
  }
  __device__ __forceinline__ int token(int row) const { return first + (row >> pack_log2); }
  __device__ __forceinline__ int head_of(int row) const { return head + (row & ((1 << pack_log2) - 1)); }
};

// The visible keys of a tile of queries: the union over its rows, and what
// all of its rows see.
struct TileKeys {
  int32_t s_end, lo, hi;             // union: [0, s_end) and [lo, hi)
  int32_t all_s_end, all_lo, all_hi; // every row sees [0, all_s_end) and [all_lo, all_hi)
  __device__ __forceinline__ TileKeys(const AttentionParams& p, const Lengths& n, int i0) {
    s_end = lo = hi = all_s_end = all_lo = all_hi = 0;
    const int i1 = min(i0 + (kTile >> p.pack_log2), n.q) - 1;
    if (i0 > i1) return;
    const Visible first = visible_keys(n.position(i0), n.kv, p.window, p.sinks);
    const Visible last = visible_keys(n.position(i1), n.kv, p.window, p.sinks);
    lo = first.lo;
    hi = last.hi;
    s_end = min(last.s_end, lo);
    all_lo = last.lo;
    all_hi = first.hi;
    all_s_end = first.s_end;
  }
  __device__ __forceinline__ bool every(int k0) const {
    return k0 + kTile <= all_s_end || (k0 >= all_lo && k0 + kTile <= all_hi);
  }
};

// A query tile's key tiles, numbered densely.
struct TileList {
  int32_t n_sink, w_beg, n;
  __device__ __forceinline__ explicit TileList(const TileKeys& a) {
    const int s = (a.s_end + kTile - 1) / kTile;
    w_beg = a.lo < a.hi ? a.lo / kTile : s;
    n_sink = min(s, w_beg);
    n = n_sink + (a.lo < a.hi ? (a.hi + kTile - 1) / kTile - w_beg : s - n_sink);
  }
  __device__ __forceinline__ int key(int j) const { return (j < n_sink ? j : j - n_sink + w_beg) * kTile; }
};

__device__ __forceinline__ uint32_t below_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Bit c: the row sees key k0 + c, 32 keys.
__device__ __forceinline__ uint32_t visible_bits32(const Visible& v, int k0) {
  return (below_bits(v.hi - k0) & ~below_bits(v.lo - k0)) | below_bits(v.s_end - k0);
}

// Zero the rows of a staged tile for which keep(row) is false: they may hold
// NaN, and 0 times NaN is NaN. One warp, 4 rows at a time.
template <int DP, typename Keep>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int lane, Keep keep) {
  tile += lane * 16;
#pragma unroll 1
  for (int r = lane >> 3; r < kTile; r += 4, tile += 512) {
    if (keep(r)) continue;
#pragma unroll
    for (int box = 0; box < DP / 64; ++box) *reinterpret_cast<uint4*>(tile + box * (kTile * 128)) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// Keys (or values) k0.. of which no query of the sequence sees some.
template <int DP>
__device__ __forceinline__ void clear_unseen(const Visible& seen, uint8_t* tile, int k0, int kv_len, int lane) {
  const int end = min(k0 + kTile, kv_len);  // the copy wrote zeros from here on
  if (end <= seen.s_end || (k0 >= seen.lo && end <= seen.hi)) return;
  clear_rows<DP>(tile, lane, [&](int r) { return sees(seen, k0 + r); });
}

// What the queries of a sequence see together.
__device__ __forceinline__ Visible sequence_keys(const AttentionParams& p, const Lengths& n) {
  Visible v{0, 0, 0};
  if (n.q > 0) {
    const Visible first = visible_keys(n.position(0), n.kv, p.window, p.sinks);
    v = visible_keys(n.position(n.q - 1), n.kv, p.window, p.sinks);
    v.lo = min(v.lo, first.lo);
    v.s_end = min(v.s_end, v.lo);
  }
  return v;
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

// Maximum of 128 scores: eight chains, so that no long one holds a row up.
__device__ __forceinline__ float max128(const uint32_t* s) {
  float m[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) m[q] = __uint_as_float(s[q]);
#pragma unroll
  for (int e = 8; e < 120; e += 16)
#pragma unroll
    for (int q = 0; q < 8; ++q) m[q] = fmaxf(fmaxf(m[q], __uint_as_float(s[e + q])), __uint_as_float(s[e + q + 8]));
#pragma unroll
  for (int q = 0; q < 8; ++q) m[q] = fmaxf(m[q], __uint_as_float(s[120 + q]));
  return fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), fmaxf(fmaxf(m[4], m[5]), fmaxf(m[6], m[7])));
}

// A row's P = 2^(sl s + nb) in 16-bit pairs to TMEM; its sum. (Taking some of the
// exponentials by a polynomial, to spare the exponential unit, was slower at
// every share from 1 to 4 in 8: 438 us at 0, 445 at 1, 468 at 2 for 16384
// queries, window 4096, dim 128. Packed f32x2 arithmetic: 438, scalar 434.)
template <typename T>
__device__ __forceinline__ float write_p(const uint32_t* s, float sl, float nb, uint32_t at) {
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t packed[16];
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      const float x = ex2(__fmaf_rn(__uint_as_float(s[c * 32 + e]), sl, nb));
      const float y = ex2(__fmaf_rn(__uint_as_float(s[c * 32 + e + 1]), sl, nb));
      sum[e & 2] += x;
      sum[(e & 2) + 1] += y;
      packed[e / 2] = T::pack(x, y);
    }
    tmem_store16(at + c * 16, packed);
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <int DP>
struct TileSmem {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kStages = DP == 128 ? 2 : 4;
  static constexpr int kBytes = (1 + kStages) * kTileBytes + 1024;  // 1024: alignment of the swizzle
};

struct TileBarriers {
  uint64_t q_full, s_full, p_full, o_full, kv_full[4], kv_empty[4];
  uint32_t tmem, gone;
};

constexpr int kTileThreads = 256;

template <typename T, int DP>
__global__ void __launch_bounds__(kTileThreads, 2) attention_tiles_kernel(const __grid_constant__ TileParams tp) {
  using Smem = TileSmem<DP>;
  constexpr int kStages = Smem::kStages, kTileBytes = Smem::kTileBytes, kBox = kTile * 128;
  constexpr uint32_t kColumns = 256;
  constexpr float kShift = T::kIsHalf ? 7.f : 0.f, kMaxLag = 8.f;
  extern __shared__ uint8_t dynamic[];
  __shared__ TileBarriers bars;
  uint8_t* q_tile = dynamic + ((1024 - (smem_addr(dynamic) & 1023)) & 1023);
  uint8_t* stages = q_tile + kTileBytes;
  const AttentionParams& p = tp.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 4 && lane == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.s_full, 1);
    mbar_init(&bars.p_full, 4);
    mbar_init(&bars.o_full, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.kv_full[i], 1);
      mbar_init(&bars.kv_empty[i], 1);
    }
    bars.gone = 0;
    fence_barrier_init();
    prefetch_map(&tp.q);
    prefetch_map(&tp.k);
    prefetch_map(&tp.v);
    prefetch_map(&tp.o);
  }
  if (warp == 5) tmem_alloc(&bars.tmem, kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem, s_tmem = tmem, o_tmem = tmem + 128;
  pdl_wait();

  const int which = p.by_heads.div(blockIdx.x), bk = blockIdx.x - which * p.by_heads.by, b = p.by_kv_heads.div(bk), hk = bk - b * p.kv_heads;
  const int unit = tp.splits == 1 ? which : which / tp.splits, split = which - unit * tp.splits;
  const QueryTile tile(p, hk, unit, tp.q_tiles);
  const Lengths len(p, b);
  const TileKeys keys(p, len, tile.first);
  const TileList list(keys);
  // This CTA's key tiles.
  int j0 = 0, n = list.n;
  if (tp.splits > 1) {
    j0 = (int)((int64_t)list.n * split / tp.splits);
    n = (int)((int64_t)list.n * (split + 1) / tp.splits) - j0;
  }
  const Waiter wait{&bars.gone, p.status, kWaitNs};

  if (warp >= 4) {
    registers_down<80>();
    if (warp == 4) {
      // ---- loads
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars.q_full, kTileBytes);
#pragma unroll
        for (int box = 0; box < DP / 64; ++box)
          tma_load(q_tile + box * kBox, &tp.q, box * 64, tile.head, tile.first, b, &bars.q_full);
        RingPos ring;
        for (int j = 0; j < 2 * n; ++j, ring.next(kStages)) {  // K and V in turn
          if (!wait(&bars.kv_empty[ring.s], ring.ph ^ 1)) break;
          mbar_arrive_expect_tx(&bars.kv_full[ring.s], kTileBytes);
#pragma unroll
          for (int box = 0; box < DP / 64; ++box)
            tma_load(stages + ring.s * kTileBytes + box * kBox, j & 1 ? &tp.v : &tp.k, box * 64, hk, list.key(j0 + (j >> 1)), b,
                     &bars.kv_full[ring.s]);
        }
      }
      __syncwarp();
    } else if (warp == 5) {
      // ---- products: S(j), then P(j) V(j) and S(j + 1), ...
      const Visible seen = sequence_keys(p, len);
      const uint32_t one = elect_one();
      auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
      RingPos ring;
      bool ok = warp_wait(&bars.q_full, 0);
      for (int j = 0; j <= n && ok; ++j) {
        const int v_slot = ring.s;
        if (j > 0) {
          if (!warp_wait(&bars.kv_full[v_slot], ring.ph)) break;
          clear_unseen<DP>(seen, stages + v_slot * kTileBytes, list.key(j0 + j - 1), p.kv_len, lane);
          ring.next(kStages);
        }
        if (j < n && !warp_wait(&bars.kv_full[ring.s], ring.ph)) break;
        if (j > 0) {
          if (!warp_wait(&bars.p_full, (j - 1) & 1)) break;
          tc_fence_after();
          mma_columns<T, DP, kTile, 32>(one, o_tmem, s_tmem, stages + v_slot * kTileBytes, kBox, j > 1);
        }
        if (j < n) {
          // One queue of products: commits come behind both (a commit between
          // them cost 7% at 16384 queries, window 4096, dim 128: 508 us, now 474).
          mma_rows<T, DP, kTile>(one, s_tmem, q_tile, kBox, stages + ring.s * kTileBytes, kBox);
          mma_commit(one, &bars.s_full);
          if (j > 0) mma_commit(one, &bars.kv_empty[v_slot]);
          mma_commit(one, &bars.kv_empty[ring.s]);
          ring.next(kStages);
        } else {
          mma_commit(one, &bars.o_full);
        }
      }
    }
  } else {
    // ---- softmax, one thread per query
    registers_up<176>();
    const int i = tile.token(threadIdx.x);
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const uint32_t s_at = s_tmem + lanes, o_at = o_tmem + lanes;
    const bool in = i < len.q;
    const Visible see = visible_keys(in ? len.position(i) : -1, len.kv, p.window, p.sinks);
    // Scale 0 would make masked scores 0 * -infinity; the least normal number
    // gives the same result for scores below 10^30.
    const float sl = fmaxf(p.scale * kLog2e, 1.1754944e-38f);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int k0 = list.key(j0 + j);
      ok = __all_sync(0xffffffffu, wait(&bars.s_full, j & 1));
      if (!ok) break;
      tc_fence_after();
      uint32_t raw[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_load32(s_at + c * 32, raw + c * 32);
      tmem_wait_loads();
      if (!keys.every(k0)) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t bits = visible_bits32(see, k0 + c * 32);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((bits >> e) & 1)) raw[c * 32 + e] = 0xFF800000u;
        }
      }
      const float top = max128(raw) * sl;
      if (__any_sync(0xffffffffu, top > m + kMaxLag)) {
        const float next = fmaxf(m, top), f = next == -INFINITY ? 1.f : ex2(m - next);
        m = next;
        l *= f;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            tmem_load32(o_at + c, o);
            tmem_wait_loads();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_store32(o_at + c, o);
          }
        }
      }
      const float nb = m == -INFINITY ? 0.f : kShift - m;
      l += write_p<T>(raw, sl, nb, s_at);
      tmem_wait_stores();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_full);
    }
    // ---- output, staged where the queries were; a part of it straight to memory
    if (ok) ok = __all_sync(0xffffffffu, wait(&bars.o_full, 0));
    const bool whole = tp.splits == 1;
    if (ok) {
      tc_fence_after();
      const float inv = !in || l == 0.f ? 0.f : l > 0.f ? rcp_rn(l) : l;  // a NaN stays one
      float4* part = reinterpret_cast<float4*>(tp.part_o) + (int64_t)blockIdx.x * (kTile * DP / 4) + threadIdx.x;
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_load32(o_at + c, o);
          tmem_wait_loads();
        }
        if (whole) {
          stage32<T>(q_tile, threadIdx.x, c, o, inv, n > 0 && inv != 0.f);
        } else if (n > 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            part[(c / 4 + e) * kTile] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                                    __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
        }
      }
      if (!whole)  // -infinity: no key seen; a NaN among the scores goes on in the sum
        reinterpret_cast<float2*>(tp.part_stats)[(int64_t)blockIdx.x * kTile + threadIdx.x] =
            make_float2(!in || l == 0.f ? -INFINITY : m == -INFINITY ? 0.f : m, l);
      else if (p.lse && i < p.q_len)
        p.lse[((int64_t)b * p.heads + tile.head_of(threadIdx.x)) * p.q_len + i] =
            !in || l == 0.f ? -INFINITY : (m - kShift + __log2f(l)) * (1.f / kLog2e);
      fence_proxy_async_smem();
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (threadIdx.x == 0 && whole && !*(volatile uint32_t*)&bars.gone) {
#pragma unroll
      for (int box = 0; box < DP / 64; ++box)
        if (box * 64 < p.head_dim) tma_store(&tp.o, q_tile + box * kBox, box * 64, tile.head, tile.first, b);
      bulk_commit();
      bulk_wait_all();
    }
  }
  finish_tmem(bars.gone, warp == 5, tmem, kColumns);
}

// Joins the CTAs of a query tile. kGroups threads take the CTAs of a row in
// turn, 4 dims each; grid.x tiles as in the kernel above, grid.y the rest of the
// rows and dims. (8 queries of 8 heads over 65536 keys, 128 CTAs a tile: 52.6 us with
// one thread a row, 27.9 with 4, 21.0 with 16; 128 over 16384, 32 CTAs: 24.8, 19.0,
// 24.2; 288 over 16384, 16 CTAs: 28.3, 28.1, 38.8.)
template <typename T, int DP, int kGroups>
__global__ void __launch_bounds__(256) attention_tiles_join_kernel(const __grid_constant__ TileParams tp) {
  constexpr float kShift = T::kIsHalf ? 7.f : 0.f;
  constexpr int kRows = kGroups == 1 ? kTile : 256 / kGroups, kQuads = 256 / kRows / kGroups;
  __shared__ float sm[kGroups == 1 ? 1 : kGroups][kRows][6];
  const AttentionParams& p = tp.a;
  const int unit = p.by_heads.div(blockIdx.x), bk = blockIdx.x - unit * p.by_heads.by, b = p.by_kv_heads.div(bk), hk = bk - b * p.kv_heads;
  const int in_cta = threadIdx.x % kRows, group = threadIdx.x / kRows % kGroups;
  const int row = blockIdx.y % (kTile / kRows) * kRows + in_cta;
  const int quad = blockIdx.y / (kTile / kRows) * kQuads + threadIdx.x / (kRows * kGroups);
  const QueryTile tile(p, hk, unit, tp.q_tiles);
  const int i = tile.token(row), h = tile.head_of(row);
  pdl_wait();
  const int64_t first = (int64_t)unit * tp.splits * p.by_heads.by + bk;  // CTA of split 0; the next is by_heads.by further
  const float2* stats = reinterpret_cast<const float2*>(tp.part_stats) + first * kTile + row;
  const float4* part = reinterpret_cast<const float4*>(tp.part_o) + first * (kTile * DP / 4) + quad * kTile + row;
  const int64_t step = (int64_t)p.by_heads.by * kTile;
  float top = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int s = group; s < tp.splits; s += kGroups) top = fmaxf(top, stats[s * step].x);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = group; s < tp.splits; s += kGroups) {
    const float2 st = stats[s * step];
    const float4 v = part[s * step * (DP / 4)];
    if (st.x == -INFINITY) continue;  // saw no key
    const float f = ex2(st.x - top);
    sum = __fmaf_rn(f, st.y, sum);
    o.x = __fmaf_rn(f, v.x, o.x);
    o.y = __fmaf_rn(f, v.y, o.y);
    o.z = __fmaf_rn(f, v.z, o.z);
    o.w = __fmaf_rn(f, v.w, o.w);
  }
  if (kGroups > 1) {
    float* mine = sm[group][in_cta];
    mine[0] = top;
    mine[1] = sum;
    mine[2] = o.x;
    mine[3] = o.y;
    mine[4] = o.z;
    mine[5] = o.w;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) top = fmaxf(top, sm[g][in_cta][0]);
    sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const float* other = sm[g][in_cta];
      if (other[0] == -INFINITY) continue;
      const float f = ex2(other[0] - top);
      sum = __fmaf_rn(f, other[1], sum);
      o.x = __fmaf_rn(f, other[2], o.x);
      o.y = __fmaf_rn(f, other[3], o.y);
      o.z = __fmaf_rn(f, other[4], o.z);
      o.w = __fmaf_rn(f, other[5], o.w);
    }
  }
  if (i >= p.q_len) return;
  const float inv = sum == 0.f ? 0.f : rcp_rn(sum);
  if (quad * 4 < p.head_dim)
    *reinterpret_cast<uint2*>(p.o.at(b, i, h) + quad * 4) = make_uint2(T::pack(o.x * inv, o.y * inv), T::pack(o.z * inv, o.w * inv));
  if (quad == 0 && p.lse)
    p.lse[((int64_t)b * p.heads + h) * p.q_len + i] = sum == 0.f ? -INFINITY : (top - kShift + __log2f(sum)) * (1.f / kLog2e);
}

}  // namespace cs
