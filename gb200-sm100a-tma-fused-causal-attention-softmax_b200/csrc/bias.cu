// C ABI of the biased causal softmax and its gradient: bucket borders,
// argument checks, launch shapes (kernels/bias.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "causal_attention.h"
#include "causal_softmax.h"
#include "internal.hpp"
#include "kernels/bias.cuh"

namespace {

using cs_host::fail;
using cs_host::fail_cuda;

constexpr int64_t kI32Max = 2147483647;

// Whole numbers of up to 1024 bits: powers of a distance (14 bits) up to the
// 64th, the most that cs_bias_buckets forms.
struct Big {
  uint32_t limb[32] = {1};
  int n = 1;
};

void multiply(Big* a, uint32_t by) {
  uint64_t carry = 0;
  for (int i = 0; i < a->n; ++i) {
    carry += (uint64_t)a->limb[i] * by;
    a->limb[i] = (uint32_t)carry;
    carry >>= 32;
  }
  if (carry) a->limb[a->n++] = (uint32_t)carry;
}

Big power(uint32_t base, int exp, Big from = Big{}) {
  for (int i = 0; i < exp; ++i) multiply(&from, base);
  return from;
}

bool less(const Big& a, const Big& b) {
  if (a.n != b.n) return a.n < b.n;
  for (int i = a.n; i-- > 0;)
    if (a.limb[i] != b.limb[i]) return a.limb[i] < b.limb[i];
  return false;
}

int check_args(const cs_bias_args* a) {
  if (!a) return fail(CS_ERR_NULL, "arguments are null");
  if (a->type != CS_TYPE_F16 && a->type != CS_TYPE_BF16) return fail(CS_ERR_ARG, "unknown element type %d", a->type);
  if (a->batch <= 0 || a->heads <= 0 || a->rows <= 0 || a->cols <= 0)
    return fail(CS_ERR_EMPTY, "batch %d, heads %d, rows %d and cols %d must be positive", a->batch, a->heads, a->rows, a->cols);
  if (a->pitch < a->cols || (a->pitch & 7)) return fail(CS_ERR_PITCH, "pitch %d for %d columns", a->pitch, a->cols);
  if (a->row_offset < 0 || a->row_offset > kI32Max - a->rows || a->pitch > kI32Max - 8)
    return fail(CS_ERR_WRONG_LENGTH, "row offset %d with %d rows", a->row_offset, a->rows);
  // The matrices' elements count in 62 bits.
  const int64_t matrices = (int64_t)a->batch * a->heads, size = (int64_t)a->rows * a->pitch;
  if (matrices > (INT64_MAX >> 1) / size)
    return fail(CS_ERR_WRONG_LENGTH, "%lld matrices of %lld elements", (long long)matrices, (long long)size);
  if (matrices > (int64_t)1 << 30) return fail(CS_ERR_WRONG_LENGTH, "%lld matrices: at most 2^30", (long long)matrices);
  if (a->window < 0 || a->sinks < 0) return fail(CS_ERR_ARG, "window %d and sinks %d must not be negative", a->window, a->sinks);
  if (!std::isfinite(a->scale) || !(a->scale >= 0.f && a->scale <= CS_MAX_SCALE))
    return fail(CS_ERR_BAD_SCALE, "scale %g", (double)a->scale);
  if (a->buckets < 1 || a->buckets > CS_MAX_BUCKETS) return fail(CS_ERR_ARG, "%d buckets: 1 to %d", a->buckets, CS_MAX_BUCKETS);
  if (!a->bucket_starts) return fail(CS_ERR_NULL, "bucket_starts is null");
  for (int j = 0; j < a->buckets; ++j) {
    const int32_t s = a->bucket_starts[j];
    if (j == 0 ? s != 0 : s <= a->bucket_starts[j - 1] || s > CS_MAX_BUCKET_START)
      return fail(CS_ERR_ARG, "bucket %d starts at %d: starts begin at 0 and ascend to at most %d", j, s, CS_MAX_BUCKET_START);
  }
  return CS_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool overlap(const void* a, const void* b, int64_t bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + (uintptr_t)bytes && y < x + (uintptr_t)bytes;
}

int check_matrices(const cs_bias_args* a, const void* x, const void* y, const void* out) {
  if (!x || !y || !out) return fail(CS_ERR_NULL, "a matrix pointer is null");
  if (!aligned16(x) || !aligned16(y) || !aligned16(out)) return fail(CS_ERR_ALIGNMENT, "matrices must be 16-byte aligned");
  const int64_t bytes = (int64_t)a->batch * a->heads * a->rows * a->pitch * 2;
  if (overlap(x, out, bytes) || overlap(y, out, bytes)) return fail(CS_ERR_ARG, "the output overlaps an input");
  return CS_OK;
}

// Launch shape: a row takes `lanes` lanes; a CTA works on block / lanes rows at
// a time, and each matrix has `ctas` CTAs. slots: vectors of a staged
// row's buffer; buffers: of a group; both 0 where rows stay in global memory.
struct Shape {
  int lanes, block, ctas, slots, buffers;
  size_t smem;
};

// Most visible 16-byte vectors a row has.
int64_t max_vectors(const cs_bias_args* a) {
  const int64_t last = std::min<int64_t>(a->cols, (int64_t)a->row_offset + a->rows);
  int64_t n = (last + 7) / 8;
  if (a->window) n = std::min<int64_t>(n, ((int64_t)a->window + 14) / 8 + ((int64_t)a->sinks + 7) / 8);
  return n;
}

// CTAs of a matrix. The launch takes rounds of resident CTAs, and a CTA the time
// of its groups' rows and of its start and end, `ends` in quarters of a row (the
// backward adds up its groups' arrays by distance). Numbers that fill whole rounds are
// the candidates, and within 5% the one with more rounds, whose CTAs end more
// evenly. Against four rounds always, at the same lanes: backward 128 x 1024^2 146 us, 152; 16 x 2048^2
// 57, 77; 24 x 257^2 8.8, 11.1; forward 16 x 2048^2 46, 55.
int ctas_per_matrix(const cs_bias_args* a, int64_t resident, int groups, int ends) {
  const int64_t matrices = (int64_t)a->batch * a->heads, most = ((int64_t)a->rows + groups - 1) / groups;
  const int64_t rounds = (matrices + resident - 1) / resident;
  int64_t turns = most, best = INT64_MAX;  // rows of a group
  for (int64_t w = rounds; w < rounds + 8; ++w) {
    const int64_t n = std::min(most, std::max<int64_t>(1, w * resident / matrices)), t = (most + n - 1) / n;
    const int64_t cost = (matrices * n + resident - 1) / resident * (4 * t + ends);
    if (best == INT64_MAX || 20 * cost <= 21 * best) turns = t;
    best = std::min(best, cost);
  }
  return (int)((most + turns - 1) / turns);
}

using Kernel = void (*)(cs::BiasParams);

template <typename T>
Kernel forward_kernel_of(int buffers) {
  return buffers == 2 ? &cs::bias_softmax_kernel<T, 2> : buffers == 1 ? &cs::bias_softmax_kernel<T, 1> : &cs::bias_softmax_kernel<T, 0>;
}

template <typename T>
Kernel backward_kernel_of(int buffers) {
  return buffers == 2 ? &cs::bias_backward_kernel<T, 2>
                      : buffers == 1 ? &cs::bias_backward_kernel<T, 1> : &cs::bias_backward_kernel<T, 0>;
}

// matrices: 1, forward; 2, backward.
Kernel kernel_of(int type, int matrices, int buffers) {
  if (matrices == 1) return type == CS_TYPE_F16 ? forward_kernel_of<cs::F16>(buffers) : forward_kernel_of<cs::BF16>(buffers);
  return type == CS_TYPE_F16 ? backward_kernel_of<cs::F16>(buffers) : backward_kernel_of<cs::BF16>(buffers);
}

// Few lanes a row keep the work that each row costs a warp (its geometry, the
// reductions, the vectors near the diagonal) shared among several rows, and
// shared memory for the groups' rows limits how few. Measured on B200 in us, lanes
// 4 / 8 / 16 / 32 / 64: forward 1024 x 128^2 28 / 32 / 43 / 74, 24 x 257^2 7.7 / 5.7 / 6.0 /
// 8.0, 1024 x 512^2 242 / 186 / 222 / 379, 128 x 1024^2 203 / 104 / 86 / 127, 64 x 2048^2
// - / - / 158 / 184 / 275, 64 x 4096^2 - / - / 566 / 536 / 697, 8 x 8192^2 - / - / 454 / 289 /
// 289; backward 1024 x 128^2 30 / 35 / 49 / 86, 24 x 257^2 9.3 / 7.9 / 8.7 / 11, 1024 x
// 512^2 416 / 252 / 239 / 418, 128 x 1024^2 186 / 182 / 113 / 139, 64 x 2048^2 - / - / 199 /
// 197 / 291, 64 x 4096^2 - / - / 1010 / 700 / 743, 8 x 8192^2 - / - / 685 / 503 / 362 (each
// group has its array by distance). 4 lanes only where rows are short and many.
// (Windows, lanes 4 / 8 / 16, forward: 144 x 759 x 2841, 615 keys seen, 183 / 162 / 150;
// 48 x 2000^2, 128 seen, 102 / 86 / 83.)
int least_lanes(int matrices, int64_t work, bool many) {
  if (work * matrices <= 32 && many) return 4;
  return work <= (matrices == 1 ? 96 : 64) ? 8 : 16;
}

// Long rows (in vectors) have one buffer a group instead of two and fewer lanes a
// row; loads are then covered by the other groups alone. One / two buffers, us:
// forward 128 x 1300^2 141 / 128, 64 x 2048^2 158 / 162, 32 x 3300^2 197 / 199, 32 x
// 4096^2 279 / 309; backward 256 x 700^2 124 / 118, 128 x 1100^2 128 / 127, 96 x 1500^2
// 164 / 179, 64 x 2048^2 197 / 210, 32 x 4096^2 356 / 409.
int buffers_of(int matrices, int64_t vectors) { return vectors > (matrices == 1 ? 192 : 96) ? 1 : 2; }

// Shared memory of a CTA at most, else more lanes a row (fewer groups): 74 KB
// leaves three CTAs an SM, 56 and 46 four (five would need 44). 32 x 4096^2 forward, one
// buffer: 46 KB 279 us, 74 KB 293; 32 x 4096^2 backward, one buffer: 74 KB 356, 56 KB 381; 96 x 1500^2
// forward, two buffers: 74 KB 130, 46 KB 160; 256 x 400^2 backward, two: 56 KB 53, 74 KB 61.
int64_t most_smem(int matrices, int buffers) {
  if (matrices == 1) return (buffers == 1 ? 46 : 74) * 1024;
  return (buffers == 1 ? 74 : 56) * 1024;
}

// matrices: 1 (scores) or 2 (probabilities and their gradient); words: fp32
// words a CTA needs besides, per group and once.
int shape_of(const cs_bias_args* a, const cs_host::Device& d, int matrices, int64_t group_words, int64_t words, Shape* shape) {
  const int64_t nv = max_vectors(a);
  Shape s{};
  s.buffers = buffers_of(matrices, nv);
  const int64_t row_bytes = nv * 16 * matrices * s.buffers;
  auto bytes = [&](int lanes) {
    const int64_t block = std::max(cs::kBiasThreads, lanes), groups = block / lanes;
    return groups * (row_bytes + group_words * 4) + (words + block / 32 * (matrices == 1 ? 4 : 2)) * 4;
  };
  const bool many = (int64_t)a->batch * a->heads * a->rows >= (int64_t)d.sms * 512;
  const int64_t work = nv + (a->pitch / 8 - nv) / 4;  // vectors that get zeros alone are less work
  s.lanes = least_lanes(matrices, work, many);
  while (s.lanes < cs::kBiasMaxThreads && bytes(s.lanes) > most_smem(matrices, s.buffers)) s.lanes *= 2;
  s.block = std::max(cs::kBiasThreads, s.lanes);
  s.slots = (int)nv;
  s.smem = (size_t)bytes(s.lanes);
  if ((int64_t)s.smem > d.max_smem) {
    s.smem -= (size_t)(s.block / s.lanes * row_bytes);
    s.slots = s.buffers = 0;
  }
  int per_sm = 0;
  const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(
      &per_sm, reinterpret_cast<const void*>(kernel_of(a->type, matrices, s.buffers)), s.block, s.smem);
  if (e != cudaSuccess) return fail_cuda(e, "bias kernels");
  const int groups = s.block / s.lanes;
  s.ctas = ctas_per_matrix(a, (int64_t)d.sms * std::max(1, per_sm), groups, matrices == 1 ? 6 : 3 * groups);
  *shape = s;
  return CS_OK;
}

// Shared-memory limits of the kernels, once per device.
int set_up(const cs_host::Device& d) {
  static std::mutex mu;
  static bool done[cs_host::kMaxDeviceIds];
  std::lock_guard<std::mutex> lock(mu);
  if (done[d.id]) return CS_OK;
  for (int type : {CS_TYPE_F16, CS_TYPE_BF16})
    for (int matrices : {1, 2})
      for (int buffers : {0, 1, 2}) {
        const void* k = reinterpret_cast<const void*>(kernel_of(type, matrices, buffers));
        cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, d.max_smem);
        if (e == cudaSuccess && buffers)  // rows bypass L1: all of it for the buffers
          e = cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return fail_cuda(e, "bias kernels");
      }
  cudaFuncAttributes fa{};
  const cudaError_t e = cudaFuncGetAttributes(&fa, reinterpret_cast<const void*>(&cs::bias_table_kernel));
  if (e != cudaSuccess) return fail_cuda(e, "bias kernels");
  done[d.id] = true;
  return CS_OK;
}

int forward_shape(const cs_bias_args* a, const cs_host::Device& d, Shape* s) {
  return shape_of(a, d, 1, 0, cs::bias_slots(a->bucket_starts[a->buckets - 1]), s);
}

int backward_shape(const cs_bias_args* a, const cs_host::Device& d, Shape* s) {
  return shape_of(a, d, 2, cs::bias_slots(a->bucket_starts[a->buckets - 1]), 0, s);
}

cs::BiasParams params_of(const cs_bias_args* a, const Shape& s) {
  cs::BiasParams p{};
  p.heads = a->heads;
  p.rows = a->rows;
  p.cols = a->cols;
  p.pitch = a->pitch;
  p.row_offset = a->row_offset;
  p.window = a->window;
  p.sinks = a->sinks;
  p.ctas = s.ctas;
  p.lanes = s.lanes;
  p.slots = s.slots;
  p.buckets = a->buckets;
  p.near = a->bucket_starts[a->buckets - 1];
  p.scale = a->scale;
  std::copy(a->bucket_starts, a->bucket_starts + a->buckets, p.starts);
  return p;
}

int grid_of(const cs_bias_args* a, const Shape& s, int64_t* grid) {
  *grid = (int64_t)a->batch * a->heads * s.ctas;
  return *grid <= kI32Max ? CS_OK : fail(CS_ERR_WRONG_LENGTH, "%lld CTAs", (long long)*grid);
}

}  // namespace

extern "C" {

int cs_bias_buckets(int32_t buckets, int32_t max_distance, int32_t* starts) {
  if (!starts) return fail(CS_ERR_NULL, "starts is null");
  if (buckets < 2 || buckets > CS_MAX_BUCKETS || max_distance <= buckets / 2 || max_distance > CS_MAX_BUCKET_START)
    return fail(CS_ERR_ARG, "%d buckets up to distance %d: 2 to %d buckets, distance above half of them and at most %d",
                buckets, max_distance, CS_MAX_BUCKETS, CS_MAX_BUCKET_START);
  const int e = buckets / 2, m = buckets - e;
  for (int j = 0; j < e; ++j) starts[j] = j;
  for (int t = 0; t < m; ++t) {
    const Big goal = power((uint32_t)e, m - t, power((uint32_t)max_distance, t));
    int32_t lo = starts[e + t - 1] + 1, hi = std::max(lo, max_distance);  // the least n in [lo, hi]
    while (lo < hi) {
      const int32_t mid = lo + (hi - lo) / 2;
      if (less(power((uint32_t)mid, m), goal)) lo = mid + 1; else hi = mid;
    }
    starts[e + t] = lo;
  }
  // Buckets pushed up one by one by those before them may pass the limit.
  if (starts[buckets - 1] > CS_MAX_BUCKET_START) return fail(CS_ERR_ARG, "the last bucket starts at %d", starts[buckets - 1]);
  return CS_OK;
}

int cs_bias_softmax(const cs_bias_args* args, const void* x, const float* table, void* p, void* stream) {
  int rc = check_args(args);
  if (!rc) rc = check_matrices(args, x, x, p);
  if (rc) return rc;
  if (!table) return fail(CS_ERR_NULL, "table is null");
  if (reinterpret_cast<uintptr_t>(table) & 3) return fail(CS_ERR_ALIGNMENT, "table must be 4-byte aligned");
  cs_host::Device d;
  rc = cs_host::current_device(&d);
  if (!rc) rc = set_up(d);
  Shape s{};
  int64_t grid = 0;
  if (!rc) rc = forward_shape(args, d, &s);
  if (!rc) rc = grid_of(args, s, &grid);
  if (rc) return rc;
  cs::BiasParams k = params_of(args, s);
  k.x = static_cast<const uint16_t*>(x);
  k.out = static_cast<uint16_t*>(p);
  k.table = table;
  const cudaError_t e = cs_host::launch(kernel_of(args->type, 1, s.buffers), dim3((unsigned)grid), s.block, s.smem, stream, k);
  return e == cudaSuccess ? CS_OK : fail_cuda(e, "biased softmax");
}

int64_t cs_bias_softmax_backward_workspace(const cs_bias_args* args) {
  int rc = check_args(args);
  cs_host::Device d;
  if (!rc) rc = cs_host::current_device(&d);
  Shape s{};
  if (!rc) rc = set_up(d);
  if (!rc) rc = backward_shape(args, d, &s);
  if (rc) return rc;
  return (int64_t)args->batch * args->heads * s.ctas * args->buckets * 4;
}

int cs_bias_softmax_backward(const cs_bias_args* args, const void* p, const void* dp, void* ds, float* dtable,
                             void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_args(args);
  if (!rc) rc = check_matrices(args, p, dp, ds);
  if (rc) return rc;
  if (!dtable || !workspace) return fail(CS_ERR_NULL, "dtable or workspace is null");
  if (!aligned16(workspace) || (reinterpret_cast<uintptr_t>(dtable) & 3))
    return fail(CS_ERR_ALIGNMENT, "workspace must be 16-byte aligned, dtable 4-byte");
  cs_host::Device d;
  rc = cs_host::current_device(&d);
  if (!rc) rc = set_up(d);
  Shape s{};
  int64_t grid = 0;
  if (!rc) rc = backward_shape(args, d, &s);
  if (!rc) rc = grid_of(args, s, &grid);
  if (rc) return rc;
  const int64_t need = grid * args->buckets * 4;
  if ((int64_t)workspace_bytes < need)
    return fail(CS_ERR_WRONG_LENGTH, "workspace of %zu bytes, %lld needed", workspace_bytes, (long long)need);
  cs::BiasParams k = params_of(args, s);
  k.x = static_cast<const uint16_t*>(p);
  k.dp = static_cast<const uint16_t*>(dp);
  k.out = static_cast<uint16_t*>(ds);
  k.partial = static_cast<float*>(workspace);
  cudaError_t e = cs_host::launch(kernel_of(args->type, 2, s.buffers), dim3((unsigned)grid), s.block, s.smem, stream, k);
  if (e != cudaSuccess) return fail_cuda(e, "biased softmax backward");
  cs::BiasReduceParams r{};
  r.partial = k.partial;
  r.dtable = dtable;
  r.batch = args->batch;
  r.heads = args->heads;
  r.ctas = s.ctas;
  r.buckets = args->buckets;
  r.by_ctas = cs::Divider::of((uint32_t)s.ctas);
  e = cs_host::launch(&cs::bias_table_kernel, dim3((unsigned)args->heads, (unsigned)((args->buckets + 31) / 32)), 1024, 0,
                      stream, r);
  return e == cudaSuccess ? CS_OK : fail_cuda(e, "bias table gradient");
}

}  // extern "C"
