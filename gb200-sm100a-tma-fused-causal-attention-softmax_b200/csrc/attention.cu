// C ABI of attention with a sliding window and sinks: argument checks and
// launches (kernels/attention*.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include <cmath>
#include <cstdint>
#include <mutex>

#include "causal_attention.h"
#include "causal_softmax.h"
#include "internal.hpp"
#include "kernels/attention_backward.cuh"
#include "kernels/attention_tiles.cuh"
#include "kernels/attention_tokens.cuh"

// Timeout bits of the attention kernels on each device (cs_attention_status).
static __device__ __align__(256) uint32_t g_attention_status[1];

namespace {

using cs_host::fail;
using cs_host::fail_cuda;

constexpr int64_t kI32Max = 2147483647;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_tensor(const char* name, const cs_tensor& t, int32_t batch, int32_t tokens, int32_t heads, int32_t dim) {
  if (!t.data) return fail(CS_ERR_NULL, "%s is null", name);
  if (!aligned16(t.data)) return fail(CS_ERR_ALIGNMENT, "%s must be 16-byte aligned", name);
  const int64_t strides[3] = {t.batch_stride, t.token_stride, t.head_stride};
  const int32_t sizes[3] = {batch, tokens, heads};
  for (int i = 0; i < 3; ++i)
    if (sizes[i] > 1 && (strides[i] < dim || (strides[i] & 7) || strides[i] >= (int64_t)1 << 38))
      return fail(CS_ERR_PITCH, "%s: stride %lld of dimension %d must be a multiple of 8, at least head_dim (%d) and below 2^38",
                  name, (long long)strides[i], i, dim);
  return CS_OK;
}

int check_args(const cs_attention_args* a) {
  if (!a) return fail(CS_ERR_NULL, "arguments are null");
  if (a->type != CS_TYPE_F16 && a->type != CS_TYPE_BF16) return fail(CS_ERR_ARG, "unknown element type %d", a->type);
  if (a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->head_dim <= 0 || a->q_len <= 0 || a->kv_len <= 0)
    return fail(CS_ERR_EMPTY, "batch %d, heads %d and %d, head_dim %d, q_len %d and kv_len %d must be positive", a->batch,
                a->heads, a->kv_heads, a->head_dim, a->q_len, a->kv_len);
  if (a->heads % a->kv_heads) return fail(CS_ERR_ARG, "%d heads over %d kv heads", a->heads, a->kv_heads);
  if ((a->head_dim & 7) || a->head_dim > CS_MAX_HEAD_DIM)
    return fail(CS_ERR_UNSUPPORTED, "head_dim %d: a multiple of 8 up to %d", a->head_dim, CS_MAX_HEAD_DIM);
  if ((int64_t)a->batch * a->heads > 1 << 20 || a->q_len > kI32Max - 1024 || a->kv_len > kI32Max - 1024)
    return fail(CS_ERR_WRONG_LENGTH, "batch %d x heads %d (at most 2^20), q_len %d, kv_len %d", a->batch, a->heads, a->q_len, a->kv_len);
  if (a->window < 0 || a->sinks < 0) return fail(CS_ERR_ARG, "window %d and sinks %d must not be negative", a->window, a->sinks);
  if (!std::isfinite(a->scale) || !(a->scale >= 0.f && a->scale <= CS_MAX_ATTENTION_SCALE))
    return fail(CS_ERR_BAD_SCALE, "scale %g: at most %g", (double)a->scale, (double)CS_MAX_ATTENTION_SCALE);
  int rc = check_tensor("q", a->q, a->batch, a->q_len, a->heads, a->head_dim);
  if (!rc) rc = check_tensor("k", a->k, a->batch, a->kv_len, a->kv_heads, a->head_dim);
  if (!rc) rc = check_tensor("v", a->v, a->batch, a->kv_len, a->kv_heads, a->head_dim);
  if (!rc) rc = check_tensor("o", a->o, a->batch, a->q_len, a->heads, a->head_dim);
  if (rc) return rc;
  for (const void* word : {(const void*)a->q_lens, (const void*)a->kv_lens, (const void*)a->lse})
    if (reinterpret_cast<uintptr_t>(word) & 3) return fail(CS_ERR_ALIGNMENT, "q_lens, kv_lens and lse must be 4-byte aligned");
  return CS_OK;
}

// Outputs overlap neither inputs nor each other; what is plainly wrong is refused.
int check_outputs(const cs_attention_args* a) {
  for (const void* in : {a->q.data, a->k.data, a->v.data})
    if (in == a->o.data) return fail(CS_ERR_ARG, "the output is an input");
  return CS_OK;
}

int check_grads(const cs_attention_args* a, const cs_attention_grads* g) {
  if (!g) return fail(CS_ERR_NULL, "gradients are null");
  if (!a->lse) return fail(CS_ERR_NULL, "lse is null");
  int rc = check_tensor("d_o", g->d_o, a->batch, a->q_len, a->heads, a->head_dim);
  if (!rc) rc = check_tensor("dq", g->dq, a->batch, a->q_len, a->heads, a->head_dim);
  if (!rc) rc = check_tensor("dk", g->dk, a->batch, a->kv_len, a->kv_heads, a->head_dim);
  if (!rc) rc = check_tensor("dv", g->dv, a->batch, a->kv_len, a->kv_heads, a->head_dim);
  return rc;
}

int check_grad_outputs(const cs_attention_args* a, const cs_attention_grads* g) {
  const void* outs[] = {g->dq.data, g->dk.data, g->dv.data};
  for (const void* in : {a->q.data, a->k.data, a->v.data, a->o.data, g->d_o.data})
    for (const void* out : outs)
      if (in == out) return fail(CS_ERR_ARG, "a gradient's tensor is an input");
  if (outs[0] == outs[1] || outs[0] == outs[2] || outs[1] == outs[2]) return fail(CS_ERR_ARG, "two gradients share a tensor");
  return CS_OK;
}

cs::Strided strided(const cs_tensor& t) {
  return cs::Strided{static_cast<uint16_t*>(t.data), t.batch_stride, t.token_stride, t.head_stride};
}

// The driver's tensor-map encoder, looked up once.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled g_encode = nullptr;

// Boxes of 64 dims x 128 (token, head) rows, 128-byte swizzle. A dimension of
// size 1 may have any stride: it gets a valid one.
int make_map(CUtensorMap* map, const cs_attention_args* a, const cs_tensor& t, int32_t tokens, int32_t heads,
             int pack_log2) {
  const cuuint64_t row = (cuuint64_t)a->head_dim * 2;
  const cuuint64_t dims[4] = {(cuuint64_t)a->head_dim, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)a->batch};
  const cuuint64_t strides[3] = {heads > 1 ? (cuuint64_t)t.head_stride * 2 : row, tokens > 1 ? (cuuint64_t)t.token_stride * 2 : row,
                                 a->batch > 1 ? (cuuint64_t)t.batch_stride * 2 : row};
  const cuuint32_t box[4] = {64, 1u << pack_log2, (cuuint32_t)cs::kTile >> pack_log2, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = g_encode(map, a->type == CS_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                              4, t.data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? CS_OK : fail(CS_ERR_CUDA, "tensor map: driver error %d", (int)r);
}

using TileKernel = void (*)(cs::TileParams);

TileKernel tile_kernel(int type, int dim) {
  if (type == CS_TYPE_F16) return dim == 64 ? &cs::attention_tiles_kernel<cs::F16, 64> : &cs::attention_tiles_kernel<cs::F16, 128>;
  return dim == 64 ? &cs::attention_tiles_kernel<cs::BF16, 64> : &cs::attention_tiles_kernel<cs::BF16, 128>;
}

template <int kGroups>
TileKernel tile_join_kernel(int type, int dim) {
  if (type == CS_TYPE_F16)
    return dim == 64 ? &cs::attention_tiles_join_kernel<cs::F16, 64, kGroups> : &cs::attention_tiles_join_kernel<cs::F16, 128, kGroups>;
  return dim == 64 ? &cs::attention_tiles_join_kernel<cs::BF16, 64, kGroups> : &cs::attention_tiles_join_kernel<cs::BF16, 128, kGroups>;
}

int tile_smem(int dim) { return dim == 64 ? cs::TileSmem<64>::kBytes : cs::TileSmem<128>::kBytes; }

using GradKernel = void (*)(cs::GradParams);

GradKernel dq_kernel(int type, int dim) {
  if (type == CS_TYPE_F16) return dim == 64 ? &cs::attention_dq_kernel<cs::F16, 64> : &cs::attention_dq_kernel<cs::F16, 128>;
  return dim == 64 ? &cs::attention_dq_kernel<cs::BF16, 64> : &cs::attention_dq_kernel<cs::BF16, 128>;
}

GradKernel dkv_kernel(int type, int dim) {
  if (type == CS_TYPE_F16) return dim == 64 ? &cs::attention_dkv_kernel<cs::F16, 64> : &cs::attention_dkv_kernel<cs::F16, 128>;
  return dim == 64 ? &cs::attention_dkv_kernel<cs::BF16, 64> : &cs::attention_dkv_kernel<cs::BF16, 128>;
}

GradKernel dkv_join_kernel(int type, int dim) {
  if (type == CS_TYPE_F16) return dim == 64 ? &cs::attention_dkv_join_kernel<cs::F16, 64> : &cs::attention_dkv_join_kernel<cs::F16, 128>;
  return dim == 64 ? &cs::attention_dkv_join_kernel<cs::BF16, 64> : &cs::attention_dkv_join_kernel<cs::BF16, 128>;
}

int dq_smem(int dim) { return dim == 64 ? cs::QuerySmem<64>::kBytes : cs::QuerySmem<128>::kBytes; }
int dkv_smem(int dim) { return dim == 64 ? cs::KeySmem<64>::kBytes : cs::KeySmem<128>::kBytes; }

// First use of a device: kernel attributes, the status word's address.
int set_up(const cs_host::Device& d, uint32_t** status) {
  static std::mutex mu;
  static uint32_t* words[cs_host::kMaxDeviceIds];
  std::lock_guard<std::mutex> lock(mu);
  if (!words[d.id]) {
    cudaError_t e = cudaSuccess;
    if (!g_encode) {
      void* f = nullptr;
      cudaDriverEntryPointQueryResult found{};
      e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
      if (e != cudaSuccess) return fail_cuda(e, "cuTensorMapEncodeTiled");
      if (found != cudaDriverEntryPointSuccess || !f) return fail(CS_ERR_DEVICE, "the driver has no cuTensorMapEncodeTiled");
      g_encode = reinterpret_cast<EncodeTiled>(f);
    }
    for (int type : {CS_TYPE_F16, CS_TYPE_BF16})
      for (int dim : {64, 128}) {
        e = cudaFuncSetAttribute(reinterpret_cast<const void*>(tile_kernel(type, dim)),
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, tile_smem(dim));
        if (e == cudaSuccess)
          e = cudaFuncSetAttribute(reinterpret_cast<const void*>(dq_kernel(type, dim)),
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, dq_smem(dim));
        if (e == cudaSuccess)
          e = cudaFuncSetAttribute(reinterpret_cast<const void*>(dkv_kernel(type, dim)),
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, dkv_smem(dim));
        if (e != cudaSuccess) return fail_cuda(e, "attention kernels");
      }
    uint32_t* w = nullptr;
    e = cudaGetSymbolAddress(reinterpret_cast<void**>(&w), g_attention_status);
    if (e != cudaSuccess) return fail_cuda(e, "attention status word");
    words[d.id] = w;
  }
  *status = words[d.id];
  return CS_OK;
}

// Heads of a group in one query tile: the largest power of two that divides the
// group, up to a tile's rows (its logarithm).
int pack_of(const cs_attention_args* a) {
  const int group = a->heads / a->kv_heads;
  int log2 = 0;
  while (log2 < 7 && group % (2 << log2) == 0) ++log2;
  return log2;
}

int params_of(const cs_attention_args* a, cs::AttentionParams* p, cs_host::Device* d) {
  int rc = cs_host::current_device(d);
  if (!rc) rc = set_up(*d, &p->status);
  if (rc) return rc;
  p->q = strided(a->q);
  p->k = strided(a->k);
  p->v = strided(a->v);
  p->o = strided(a->o);
  p->lse = a->lse;
  p->q_lens = a->q_lens;
  p->kv_lens = a->kv_lens;
  p->batch = a->batch;
  p->heads = a->heads;
  p->kv_heads = a->kv_heads;
  p->group = a->heads / a->kv_heads;
  p->head_dim = a->head_dim;
  p->q_len = a->q_len;
  p->kv_len = a->kv_len;
  p->window = a->window;
  p->sinks = a->sinks;
  p->scale = a->scale;
  p->pack_log2 = pack_of(a);
  p->by_heads = cs::Divider::of((uint32_t)(a->batch * a->kv_heads));
  p->by_kv_heads = cs::Divider::of((uint32_t)a->kv_heads);
  p->by_packs = cs::Divider::of((uint32_t)(p->group >> p->pack_log2));
  return CS_OK;
}

int check_workspace(const void* workspace, size_t bytes, int64_t need) {
  if (need == 0) return CS_OK;
  if (!workspace) return fail(CS_ERR_NULL, "workspace is null, %lld bytes needed", (long long)need);
  if (!aligned16(workspace)) return fail(CS_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  if ((int64_t)bytes < need) return fail(CS_ERR_WRONG_LENGTH, "workspace of %zu bytes, %lld needed", bytes, (long long)need);
  return CS_OK;
}

// Few queries: the kernel for single tokens. Its launch shape.
struct TokenShape {
  int rows, dim, splits;  // rows: 8 or 16
  int64_t ctas;
  int64_t part_bytes, stats_bytes;
};

constexpr int64_t kTokenKeys = 128;    // of a CTA, at least: 2 steps a warp
constexpr int kTokenResident[2][2] = {{4, 3}, {3, 2}};  // CTAs an SM: dim 64, 128; 8, 16 rows

// Which calls those are, by the rows of a kv head, (query, head) pairs, and by the
// kv heads. Up to 8 rows: all. Up to 16, whose accumulators leave the kernel two
// CTAs an SM: while the kv heads are fewer than the SMs, so that their keys are
// split (4 x 2 queries over 16384 keys, 32 heads over 4, dim 128: 34.4 us, tiles
// 39.0; 64 x 2 over 4096: 108.7, tiles 91.8). Groups that are no power of two, whose
// tiles read the keys more than once, would gain by it there too: 64 x 1 of 48 heads
// over 4, 4096 keys: 108, by the rule's tiles 262. More rows would read the keys more
// than once (8 x 8 over 1024: 13.0, tiles 9.4).
bool few_queries(const cs_attention_args* a, int sms) {
  const int64_t rows = (int64_t)a->q_len * (a->heads / a->kv_heads);
  return rows <= 8 || (rows <= 16 && (int64_t)a->batch * a->kv_heads < sms);
}

TokenShape token_shape(const cs_attention_args* a, int sms) {
  TokenShape s{};
  const int64_t rows = (int64_t)a->q_len * (a->heads / a->kv_heads);
  s.rows = rows <= 8 ? 8 : 16;
  s.dim = a->head_dim <= 64 ? 64 : 128;
  const int64_t base = (int64_t)a->batch * a->kv_heads;
  int64_t keys = a->kv_len;
  if (a->window) keys = std::min<int64_t>(keys, (int64_t)a->window + a->q_len + a->sinks + 32);
  // Rounds of resident CTAs times a CTA's time, in keys: a CTA starts and ends in
  // the time of about 150. Splits that fill whole rounds are the candidates.
  // (64 tokens of 32 heads over 4, 4096 keys: 5 splits 89.5 us, 7 97.3, 2 114; 16
  // tokens, 8 kv heads: 3 splits 46.2, 4 60.4, 14 55.8.)
  const int64_t wave = (int64_t)sms * kTokenResident[s.dim == 128][s.rows == 16];
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(keys / kTokenKeys, cs::kMaxSplits));
  int64_t splits = 1, best = INT64_MAX;
  const int64_t rounds = (base + wave - 1) / wave;
  for (int64_t w = rounds; w < rounds + 8; ++w) {
    const int64_t n = std::min(most, std::max<int64_t>(1, w * wave / base));
    const int64_t cost = (base * n + wave - 1) / wave * (keys / n + 150);
    if (cost < best) best = cost, splits = n;
  }
  s.splits = (int)splits;
  s.ctas = base * s.splits;
  if (s.splits > 1) {
    s.part_bytes = s.ctas * s.rows * s.dim * 4;
    s.stats_bytes = s.ctas * s.rows * 8;
  }
  return s;
}

using TokenKernel = void (*)(cs::TokenParams);

template <typename T>
TokenKernel token_kernel_of(int dim, int rows) {
  if (dim == 64) return rows == 8 ? &cs::attention_tokens_kernel<T, 64, 1> : &cs::attention_tokens_kernel<T, 64, 2>;
  return rows == 8 ? &cs::attention_tokens_kernel<T, 128, 1> : &cs::attention_tokens_kernel<T, 128, 2>;
}

int launch_tokens(const cs_attention_args* a, const cs::AttentionParams& p, const TokenShape& s, void* workspace, void* stream) {
  cs::TokenParams t{};
  t.a = p;
  t.part_o = static_cast<float*>(workspace);
  t.part_stats = reinterpret_cast<float*>(static_cast<char*>(workspace) + s.part_bytes);
  t.splits = s.splits;
  t.rows = s.rows;
  t.dim_pad = s.dim;
  if (s.ctas * s.rows > kI32Max) return fail(CS_ERR_WRONG_LENGTH, "%lld CTAs", (long long)s.ctas);
  const bool half = a->type == CS_TYPE_F16;
  cudaError_t e = cs_host::launch(half ? token_kernel_of<cs::F16>(s.dim, s.rows) : token_kernel_of<cs::BF16>(s.dim, s.rows),
                                  dim3((unsigned)s.ctas), cs::kTokenWarps * 32, 0, stream, t);
  if (e != cudaSuccess) return fail_cuda(e, "attention, few queries");
  if (s.splits == 1) return CS_OK;
  const dim3 rows((unsigned)((int64_t)a->batch * a->heads * a->q_len));
  if (s.splits > 16)
    e = cs_host::launch(half ? &cs::attention_join_kernel<cs::F16, 16> : &cs::attention_join_kernel<cs::BF16, 16>, rows, 512, 0, stream, t);
  else
    e = cs_host::launch(half ? &cs::attention_join_kernel<cs::F16, 4> : &cs::attention_join_kernel<cs::BF16, 4>, rows, 128, 0, stream, t);
  return e == cudaSuccess ? CS_OK : fail_cuda(e, "attention, joining the splits");
}

// Query tiles and, where they are too few for the SMs, the CTAs that share one's
// keys. Below 16 key tiles one CTA an SM and none split below 5: a CTA takes
// about 2 us a key tile and joining 3 (64 queries over 1100 keys, 8 heads of one
// kv head: 9 CTAs a tile 13.0 us, 1 22.1; 4096 queries, 4 heads, window 1024, two
// CTAs an SM: 23.1, one 19.6). From 16 on two an SM with at least 4 key tiles
// each (1 x 2000, 4 heads: 16.6 us, one an SM 21.0; 8 x 17 queries over 4096: 18.3
// us, with 3 key tiles 24.9).
struct TileShape {
  int dim, q_tiles, splits;
  int64_t ctas, part_bytes, stats_bytes;
};

TileShape tile_shape(const cs_attention_args* a, int sms) {
  TileShape s{};
  s.dim = a->head_dim <= 64 ? 64 : 128;
  const int pack = pack_of(a), tokens = cs::kTile >> pack;
  s.q_tiles = (a->q_len + tokens - 1) / tokens;
  const int64_t base = (int64_t)a->batch * (a->heads >> pack) * s.q_tiles;
  int64_t keys = ((int64_t)a->kv_len + cs::kTile - 1) / cs::kTile;
  if (a->window)
    keys = std::min(keys, ((int64_t)a->window + tokens + cs::kTile - 1) / cs::kTile + ((int64_t)a->sinks + cs::kTile - 1) / cs::kTile);
  const bool few = keys < 16;
  s.splits = keys < 5 ? 1 : (int)std::max<int64_t>(1, std::min((few ? 1 : 2) * (int64_t)sms / base, few ? keys : keys / 4));
  s.ctas = base * s.splits;
  if (s.splits > 1) {
    s.part_bytes = s.ctas * cs::kTile * s.dim * 4;
    s.stats_bytes = s.ctas * cs::kTile * 8;
  }
  return s;
}

int launch_tiles(const cs_attention_args* a, const cs::AttentionParams& p, const TileShape& s, void* workspace, void* stream) {
  cs::TileParams t{};
  t.a = p;
  t.q_tiles = s.q_tiles;
  t.splits = s.splits;
  t.part_o = static_cast<float*>(workspace);
  t.part_stats = reinterpret_cast<float*>(static_cast<char*>(workspace) + s.part_bytes);
  int rc = make_map(&t.q, a, a->q, a->q_len, a->heads, p.pack_log2);
  if (!rc) rc = make_map(&t.k, a, a->k, a->kv_len, a->kv_heads, 0);
  if (!rc) rc = make_map(&t.v, a, a->v, a->kv_len, a->kv_heads, 0);
  if (!rc) rc = make_map(&t.o, a, a->o, a->q_len, a->heads, p.pack_log2);
  if (rc) return rc;
  if (s.ctas > kI32Max) return fail(CS_ERR_WRONG_LENGTH, "%lld CTAs", (long long)s.ctas);
  cudaError_t e = cs_host::launch(tile_kernel(a->type, s.dim), dim3((unsigned)s.ctas), cs::kTileThreads, (size_t)tile_smem(s.dim),
                                  stream, t);
  if (e != cudaSuccess) return fail_cuda(e, "attention, tiles");
  if (s.splits == 1) return CS_OK;
  const unsigned tiles = (unsigned)(s.ctas / s.splits), dims = (unsigned)s.dim;
  if (s.splits > 64)
    e = cs_host::launch(tile_join_kernel<16>(a->type, s.dim), dim3(tiles, 2 * dims), 256, 0, stream, t);
  else if (s.splits > 8)
    e = cs_host::launch(tile_join_kernel<4>(a->type, s.dim), dim3(tiles, dims / 2), 256, 0, stream, t);
  else
    e = cs_host::launch(tile_join_kernel<1>(a->type, s.dim), dim3(tiles, dims / 8), 256, 0, stream, t);
  return e == cudaSuccess ? CS_OK : fail_cuda(e, "attention, joining the splits");
}

// The backward's launch shapes and workspace.
struct GradShape {
  int dim, q_tiles, k_tiles;
  int64_t q_pad;  // rows of a pack of heads
  int share, window_shares, sink_tiles, sink_shares;
  int64_t dkv_ctas;
  int query_blocks, key_blocks;  // fp16: of 64, whose largest norms are kept
  // An array of rows (lse2, delta; fp16: |d_o|), those norms and dQ's counter.
  int64_t rows_bytes, query_bytes, key_bytes, partial_bytes;
  int64_t counter_at() const { return (query_bytes ? 3 : 2) * rows_bytes + query_bytes + key_bytes; }
  int64_t partial_at() const { return counter_at() + 16; }
  int64_t bytes() const { return partial_at() + partial_bytes; }
};

// A key tile's work is its units, the query tiles that see it. Tiles are cut into shares
// only where that evens out the SMs: the sinks' tile, which every query sees,
// and tiles of long rows when there are few of them; each share costs a part of
// dK and dV in fp32, written and read once more. So: about two shares an SM of at least
// 16 units, fewer units only if those would not be two an SM, and no cut of a
// window's tiles as long as that makes them at most twice as long. (Training step,
// at least 16 units / this: 4 x 236 tokens, 8 heads over 1: 47.1 / 31.3 us; 5 x 149, 16
// over 2: 36.9 / 29.9. With one share an SM 2048 tokens, 8 heads over 1, took 80.3 us,
// this 68.3.)
GradShape grad_shape(const cs_attention_args* a, int sms) {
  GradShape s{};
  s.dim = a->head_dim <= 64 ? 64 : 128;
  const int pack = pack_of(a), tokens = cs::kTile >> pack;
  s.q_tiles = (a->q_len + tokens - 1) / tokens;
  s.q_pad = (int64_t)s.q_tiles * cs::kTile;
  s.k_tiles = (a->kv_len + cs::kTile - 1) / cs::kTile;
  const int64_t packs = (a->heads / a->kv_heads) >> pack, heads = (int64_t)a->batch * a->kv_heads;
  const int64_t all = s.q_tiles * packs;  // units of a tile that every query sees
  int64_t usual = all;
  if (a->window) {
    usual = std::min(all, (((int64_t)a->window + cs::kTile + tokens - 2) / tokens + 1) * packs);
    s.sink_tiles = (int)std::min<int64_t>(s.k_tiles, ((int64_t)a->sinks + cs::kTile - 1) / cs::kTile);
  }
  // Without a window tiles see half of the queries on average.
  const int64_t mean = usual < all ? usual : (usual + 1) / 2;
  const int64_t total = heads * (s.sink_tiles * all + (s.k_tiles - s.sink_tiles) * mean);
  const int64_t least = std::min<int64_t>(16, std::max<int64_t>(2, (2 * total + sms - 1) / sms));
  int64_t share = std::max(least, (total + 2 * sms - 1) / (2 * sms));
  if (usual <= 2 * share) share = std::max(share, usual);
  s.share = (int)std::min(share, std::max(all, usual));
  s.window_shares = (int)((usual + s.share - 1) / s.share);
  s.sink_shares = (int)((all + s.share - 1) / s.share);
  s.dkv_ctas = heads * ((int64_t)s.sink_tiles * s.sink_shares + (int64_t)(s.k_tiles - s.sink_tiles) * s.window_shares);
  s.rows_bytes = (int64_t)a->batch * (a->heads >> pack) * s.q_pad * 4;
  if (a->type == CS_TYPE_F16) {
    s.query_blocks = (int)((s.q_pad >> pack) + cs::kRowsPerCta - 1) / cs::kRowsPerCta;
    s.key_blocks = 2 * s.k_tiles;
    s.query_bytes = ((int64_t)a->batch * a->heads * s.query_blocks * 8 + 15) / 16 * 16;
    s.key_bytes = (heads * s.key_blocks * 4 + 15) / 16 * 16;
  }
  if (s.window_shares > 1 || (s.sink_tiles && s.sink_shares > 1)) s.partial_bytes = s.dkv_ctas * 2 * cs::kTile * s.dim * 4;
  return s;
}

int check_shape(const cs_attention_args* a, const GradShape& s) {
  if (s.q_pad > kI32Max || s.dkv_ctas > kI32Max || (int64_t)a->batch * a->heads * s.q_tiles > kI32Max - 65536)
    return fail(CS_ERR_WRONG_LENGTH, "backward of q_len %d, kv_len %d: too many tiles", a->q_len, a->kv_len);
  return CS_OK;
}

int launch_backward(const cs_attention_args* a, const cs_attention_grads* g, const cs::AttentionParams& p, const GradShape& s,
                    int sms, void* workspace, void* stream) {
  char* at = static_cast<char*>(workspace);
  float* lse2 = reinterpret_cast<float*>(at);
  float* delta = reinterpret_cast<float*>(at + s.rows_bytes);
  float* grad_norms = reinterpret_cast<float*>(at + 2 * s.rows_bytes);
  float2* grad_tops = reinterpret_cast<float2*>(at + 3 * s.rows_bytes);
  float* value_tops = reinterpret_cast<float*>(at + 3 * s.rows_bytes + s.query_bytes);
  const bool half = a->type == CS_TYPE_F16;

  cs::RowsParams r{};
  r.a = p;
  r.lse2 = lse2;
  r.delta = delta;
  r.grad_norms = grad_norms;
  r.grad_tops = grad_tops;
  r.value_tops = value_tops;
  r.next = reinterpret_cast<int32_t*>(at + s.counter_at());
  r.q_pad = (int32_t)s.q_pad;
  r.query_blocks = s.query_blocks;
  r.key_blocks = s.key_blocks;
  const unsigned rows = (unsigned)(((s.q_pad >> p.pack_log2) + cs::kRowsPerCta - 1) / cs::kRowsPerCta + s.key_blocks);
  cudaError_t e = cs_host::launch(half ? &cs::attention_rows_kernel<cs::F16> : &cs::attention_rows_kernel<cs::BF16>,
                      dim3(rows, (unsigned)std::min(a->batch * a->heads, 65535)), 256, 0, stream, r);
  if (e != cudaSuccess) return fail_cuda(e, "attention backward, rows");

  cs::GradParams k{};
  k.a = p;
  k.lse2 = lse2;
  k.delta = delta;
  k.grad_norms = grad_norms;
  k.grad_tops = grad_tops;
  k.value_tops = value_tops;
  k.query_blocks = s.query_blocks;
  k.key_blocks = s.key_blocks;
  k.next = r.next;
  k.partial = reinterpret_cast<float*>(at + s.partial_at());
  k.q_pad = (int32_t)s.q_pad;
  k.share = s.share;
  k.window_shares = s.window_shares;
  k.sink_tiles = s.sink_tiles;
  k.sink_shares = s.sink_shares;
  k.tiles = s.k_tiles;
  int rc = make_map(&k.q, a, a->q, a->q_len, a->heads, p.pack_log2);
  if (!rc) rc = make_map(&k.d_o, a, g->d_o, a->q_len, a->heads, p.pack_log2);
  if (!rc) rc = make_map(&k.k, a, a->k, a->kv_len, a->kv_heads, 0);
  if (!rc) rc = make_map(&k.v, a, a->v, a->kv_len, a->kv_heads, 0);
  if (!rc) rc = make_map(&k.out0, a, g->dk, a->kv_len, a->kv_heads, 0);
  if (!rc) rc = make_map(&k.out1, a, g->dv, a->kv_len, a->kv_heads, 0);
  if (rc) return rc;
  e = cs_host::launch(dkv_kernel(a->type, s.dim), dim3((unsigned)s.dkv_ctas), cs::kGradThreads, (size_t)dkv_smem(s.dim), stream, k);
  if (e != cudaSuccess) return fail_cuda(e, "attention backward, keys");

  cs::GradParams q = k;
  q.tiles = s.q_tiles;
  rc = make_map(&q.out0, a, g->dq, a->q_len, a->heads, p.pack_log2);
  if (rc) return rc;
  q.units = (int)((int64_t)a->batch * (a->heads >> p.pack_log2) * s.q_tiles);
  e = cs_host::launch(dq_kernel(a->type, s.dim), dim3((unsigned)std::min(q.units, sms)), cs::kGradThreads, (size_t)dq_smem(s.dim),
                      stream, q);
  if (e != cudaSuccess) return fail_cuda(e, "attention backward, queries");
  if (s.partial_bytes) {
    const int64_t tiles = (int64_t)a->batch * a->kv_heads * (s.window_shares > 1 ? s.k_tiles : s.sink_tiles);
    e = cs_host::launch(dkv_join_kernel(a->type, s.dim), dim3((unsigned)tiles, 32), 256, 0, stream, k);
  }
  return e == cudaSuccess ? CS_OK : fail_cuda(e, "attention backward, joining the shares");
}

}  // namespace

extern "C" {

int64_t cs_attention_workspace(const cs_attention_args* args) {
  int rc = check_args(args);
  cs_host::Device d;
  if (!rc) rc = cs_host::current_device(&d);
  if (rc) return rc;
  if (few_queries(args, d.sms)) {
    const TokenShape s = token_shape(args, d.sms);
    return s.part_bytes + s.stats_bytes;
  }
  const TileShape s = tile_shape(args, d.sms);
  return s.part_bytes + s.stats_bytes;
}

int cs_attention(const cs_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_args(args);
  if (!rc) rc = check_outputs(args);
  if (rc) return rc;
  cs::AttentionParams p{};
  cs_host::Device d;
  rc = params_of(args, &p, &d);
  if (rc) return rc;
  if (few_queries(args, d.sms)) {
    const TokenShape s = token_shape(args, d.sms);
    rc = check_workspace(workspace, workspace_bytes, s.part_bytes + s.stats_bytes);
    return rc ? rc : launch_tokens(args, p, s, workspace, stream);
  }
  const TileShape s = tile_shape(args, d.sms);
  rc = check_workspace(workspace, workspace_bytes, s.part_bytes + s.stats_bytes);
  return rc ? rc : launch_tiles(args, p, s, workspace, stream);
}

int64_t cs_attention_backward_workspace(const cs_attention_args* args) {
  int rc = check_args(args);
  cs_host::Device d;
  if (!rc) rc = cs_host::current_device(&d);
  if (rc) return rc;
  const GradShape s = grad_shape(args, d.sms);
  rc = check_shape(args, s);
  return rc ? rc : s.bytes();
}

int cs_attention_backward(const cs_attention_args* args, const cs_attention_grads* grads, void* workspace,
                          size_t workspace_bytes, void* stream) {
  int rc = check_args(args);
  if (!rc) rc = check_grads(args, grads);
  if (!rc) rc = check_workspace(workspace, workspace_bytes, 16);
  if (!rc) rc = check_grad_outputs(args, grads);
  if (rc) return rc;
  cs::AttentionParams p{};
  cs_host::Device d;
  rc = params_of(args, &p, &d);
  if (rc) return rc;
  const GradShape s = grad_shape(args, d.sms);
  rc = check_shape(args, s);
  if (!rc) rc = check_workspace(workspace, workspace_bytes, s.bytes());
  if (rc) return rc;
  p.d_o = strided(grads->d_o);
  p.dk = strided(grads->dk);
  p.dv = strided(grads->dv);
  return launch_backward(args, grads, p, s, d.sms, workspace, stream);
}

int cs_attention_status(uint32_t* status, void* stream) {
  if (!status) return fail(CS_ERR_NULL, "status is null");
  cs_host::Device d;
  uint32_t* word = nullptr;
  int rc = cs_host::current_device(&d);
  if (!rc) rc = set_up(d, &word);
  if (rc) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t bits = 0;
  cudaError_t e = cudaMemcpyAsync(&bits, word, sizeof bits, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaMemsetAsync(word, 0, sizeof bits, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return fail_cuda(e, "attention status");
  *status = bits;
  return cs_status_error(bits);
}

}  // extern "C"
