// Attention with a sliding window and sinks: what every kernel of it shares.
#pragma once

#include "common.cuh"
#include "divider.cuh"
#include "positions.cuh"
#include "types.cuh"

namespace cs {

constexpr uint64_t kWaitNs = 2000000000ull;  // bound on a device-side wait: 2 s of GPU time

struct Strided {  // [batch, token, head, dim], element strides, dim contiguous
  uint16_t* data;
  int64_t batch, token, head;
  __device__ __forceinline__ uint16_t* at(int b, int t, int h) const {
    return data + b * batch + t * token + h * head;
  }
};

struct AttentionParams {
  Strided q, k, v, o;       // o: output; backward: the forward's output
  Strided d_o, dk, dv;      // backward (dq is written through its map)
  float* lse;               // [batch, heads, q_len]
  const int32_t* q_lens;
  const int32_t* kv_lens;
  uint32_t* status;
  int32_t batch, heads, kv_heads, group, head_dim, q_len, kv_len, window, sinks;
  int32_t pack_log2;  // query tiles: heads of a group that share a tile, as a power of two
  Divider by_heads, by_kv_heads, by_packs;  // batch * kv_heads; kv_heads; group / pack
  float scale;
};

// One sequence's lengths, clipped to the tensors.
struct Lengths {
  int32_t q, kv;
  __device__ __forceinline__ Lengths(const AttentionParams& p, int b) {
    q = p.q_lens ? min(max(p.q_lens[b], 0), p.q_len) : p.q_len;
    kv = p.kv_lens ? min(max(p.kv_lens[b], 0), p.kv_len) : p.kv_len;
  }
  // Position of query i: the queries are the sequence's last tokens.
  __device__ __forceinline__ int32_t position(int i) const { return kv - q + i; }
};

}  // namespace cs
