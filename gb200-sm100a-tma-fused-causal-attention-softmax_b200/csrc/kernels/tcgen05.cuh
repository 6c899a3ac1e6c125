// 5th-generation tensor core, tensor memory (TMEM) and tensor-map copies
// (sm_100a), as the attention kernels use them: one CTA per product
// (cta_group::1), 16-bit operands in 128-byte-swizzled shared memory or TMEM,
// fp32 accumulators in TMEM.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "common.cuh"

namespace cs {

// A wait that every role of a CTA may give up together: the first to run out
// of time reports it and raises `gone`, which ends the others' waits.
struct Waiter {
  volatile uint32_t* gone;  // shared
  uint32_t* status;         // global
  uint64_t timeout_ns;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
    if (mbar_try_wait_parity(bar, parity)) return true;
    const uint64_t start = global_timer_ns();
    while (!*gone) {
      if (mbar_try_wait_parity_sleep(bar, parity, 100000u)) return true;
      if (global_timer_ns() - start > timeout_ns) {
        *gone = 1u;
        atomicOr(status, kStatusTimeout);
      }
    }
    return false;
  }
};

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// One box of a [batch, token, head, dim] tensor: dims from d, one head, tokens
// from t on. Out-of-range elements arrive as zeros and are not stored.
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int d, int head, int t, int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(smem_addr(dst)), "l"(map), "r"(d), "r"(head), "r"(t), "r"(b), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void tma_store(const CUtensorMap* map, const void* src, int d, int head, int t, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(map),
               "r"(d), "r"(head), "r"(t), "r"(b), "r"(smem_addr(src))
               : "memory");
}

// Registers per thread of a warpgroup from here on (all its warps call it).
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// ---- TMEM

__device__ __forceinline__ void tmem_alloc(uint32_t* where, uint32_t columns) {  // one warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(where)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}

__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {  // the same warp
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this thread's lane (a warp reads the 32 lanes of its quarter).
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
}

__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// End of a kernel that holds TMEM, all threads: after a wait was given up,
// time for copies and products in flight before their memory goes.
__device__ __forceinline__ void finish_tmem(volatile uint32_t& gone, bool owner, uint32_t at, uint32_t columns) {
  tc_fence_before();
  __syncthreads();
  pdl_trigger();
  if (gone) {
    const uint64_t start = global_timer_ns();
    while (global_timer_ns() - start < 1000000ull) {}
    __syncthreads();
  }
  if (owner) {
    tc_fence_after();
    tmem_free(at, columns);
  }
}

// ---- products

// Shared-memory operand of 64-element (128-byte) rows, 128-byte swizzle, 8-row
// groups 1024 bytes apart. Summed over the contiguous dimension ("K-major"):
// the second stride is unused. Summed over the rows ("MN-major"): `apart` is
// the distance of the next 64 columns.
__device__ __forceinline__ uint64_t operand(const void* tile, uint32_t apart = 16) {
  return (uint64_t)((smem_addr(tile) >> 4) & 0x3FFF) | (uint64_t)(apart >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// fp32 accumulator, both operands fp16 or both bf16, M x N; b_rows: B is MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t product(int m, int n, bool b_rows) {
  const uint32_t type = T::kIsHalf ? 0u : 1u;
  return 1u << 4 | type << 7 | type << 10 | (b_rows ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}

// Products and commits are called by a whole converged warp, so that their
// operands are computed once per warp, and issued by the lane with `one` set.
// (Called under a branch on the lane, a product took 65 to 80 cycles to issue.)
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(what),
      "r"((uint32_t)add), "r"(one)
      : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(what),
      "r"((uint32_t)add), "r"(one)
      : "memory");
}

// Arrive on `bar` once every product issued so far by that lane is done.
__device__ __forceinline__ void mma_commit(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)), "r"(one)
      : "memory");
}

// D[128, N] (+)= A[128, DP] B[N, DP]^T, both K-major tiles of DP / 64 boxes
// (rows x 64 elements; box strides in bytes).
template <typename T, int DP, int N>
__device__ __forceinline__ void mma_rows(uint32_t one, uint32_t d, const uint8_t* a, int a_box, const uint8_t* b, int b_box) {
  const uint64_t a0 = operand(a), b0 = operand(b);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
    mma_ss(one, d, a0 + (k >> 2) * (a_box >> 4) + (k & 3) * 2, b0 + (k >> 2) * (b_box >> 4) + (k & 3) * 2,
           product<T>(128, N, false), k > 0);
}

// D[128, DP] (+)= A[128, K] B[K, DP]: A in TMEM, two elements a column, its
// 64-element parts PART columns apart (32: contiguous); B a row tile of DP / 64
// boxes.
template <typename T, int DP, int K, int PART>
__device__ __forceinline__ void mma_columns(uint32_t one, uint32_t d, uint32_t a, const uint8_t* b, int b_box, bool add) {
  const uint64_t b0 = operand(b, (uint32_t)b_box);
#pragma unroll
  for (int k = 0; k < K / 16; ++k)
    mma_ts(one, d, a + (k >> 2) * PART + (k & 3) * 8, b0 + k * (2048 >> 4), product<T>(128, DP, true), add || k > 0);
}

}  // namespace cs
