/*
 * causal_attention.h — C ABI of the operators beside the causal softmax
 * (causal_softmax.h): a causal softmax with a learned relative-position bias
 * and its gradient, and fused attention with a sliding window and a few first
 * tokens that stay visible ("sinks"), for prompts, for single tokens reading
 * a cache, and for training.
 *
 * The positional mask, the same everywhere: a query at absolute position p
 * sees key k when
 *
 *     0 <= k <= p  and  k < keys  and  (window == 0 or p - k < window or k < sinks).
 *
 * window 0 means no window (then sinks change nothing); window 1 is the
 * query's own key. A query that sees no key has probabilities +0.0, an output
 * of zeros, a log-sum-exp of -infinity and gradients of zero.
 *
 * Conventions as in causal_softmax.h: device pointers of the current device,
 * 16-byte aligned (fp32 and int32 arrays: 4-byte); outputs overlap neither
 * inputs nor each other; `stream` is a cudaStream_t as void*; functions return 0 or
 * a CS_ERR_* code (text in cs_last_error_detail), launch asynchronously,
 * allocate nothing, and keep nothing between calls; workspaces are the
 * caller's, need no initialisation, and may be reused once the call's work on
 * the stream is done (two calls that may overlap need two). Results do not
 * depend on timing: the same inputs give the same bits. The first call of a
 * kind on a device sets the kernels up; make it before a stream capture.
 * No counterpart in the reference project.
 */
#ifndef CAUSAL_ATTENTION_H
#define CAUSAL_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of matrices, queries, keys, values and their gradients. */
enum { CS_TYPE_F16 = 0, CS_TYPE_BF16 = 1 };

/* ---------------------------------------------------------------- */
/* Causal softmax with a bias learned per bucket of distances        */
/* ---------------------------------------------------------------- */

#define CS_MAX_BUCKETS 128
#define CS_MAX_BUCKET_START 8192 /* largest first distance of a bucket */

/* First distance of each bucket (host query): half of the buckets hold one
 * distance each, the rest grow by an even ratio up to max_distance, and the
 * last holds everything from its start on. With e = buckets / 2 and
 * m = buckets - e, bucket e + t starts at the least whole n, above the bucket
 * before, with (n / e)^m >= (max_distance / e)^t, decided in whole numbers.
 * Needs 2 <= buckets <= CS_MAX_BUCKETS and
 * buckets / 2 < max_distance <= CS_MAX_BUCKET_START. */
int cs_bias_buckets(int32_t buckets, int32_t max_distance, int32_t *starts);

/* `batch` x `heads` score matrices, matrix (b, h) at element
 * (b * heads + h) * rows * pitch; local row i is position row_offset + i and
 * its columns are keys 0..cols-1. pitch >= cols, a multiple of 8. */
typedef struct cs_bias_args {
    int32_t type;                 /* CS_TYPE_* of the matrices */
    int32_t batch, heads, rows, cols, pitch;
    int32_t row_offset;
    int32_t window, sinks;
    int32_t buckets;              /* 1..CS_MAX_BUCKETS */
    const int32_t *bucket_starts; /* host, [buckets]: 0 first, ascending, <= CS_MAX_BUCKET_START */
    float scale;                  /* finite, in [0, CS_MAX_SCALE] */
} cs_bias_args;

/* p = softmax over the visible keys of scale * x + table[head, bucket(position
 * - key)]; every other column of the row, padding included, +0.0. The table
 * is fp32, [heads, buckets]. Arithmetic is binary32, and binary64 relative to
 * the row's largest score where biased scores reach 90000 in magnitude, so that
 * finite ones stay finite up to the ends of their types (a mask of the lowest
 * value). x and p must not overlap. A row whose visible scores are all -infinity is
 * all zeros; one with a NaN or +infinity among them is NaN. */
int cs_bias_softmax(const cs_bias_args *args, const void *x, const float *table, void *p, void *stream);

/* From probabilities p and their gradient dp: dz = p (dp - sum p dp) over the
 * visible keys, ds = scale dz in the matrices' type (every other column +0.0),
 * dtable[h, j] = sum of dz over the batch, the rows and the keys of bucket j,
 * fp32, [heads, buckets]. What lies at keys that a row does not see is not
 * used. ds must overlap neither input. `workspace`: at least
 * cs_bias_softmax_backward_workspace bytes. */
int64_t cs_bias_softmax_backward_workspace(const cs_bias_args *args);
int cs_bias_softmax_backward(const cs_bias_args *args, const void *p, const void *dp, void *ds,
                             float *dtable, void *workspace, size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------- */
/* Attention with a sliding window and sinks                         */
/* ---------------------------------------------------------------- */

/* A tensor [batch, tokens, heads, head_dim]: element strides of the first
 * three (positive multiples of 8 wherever that size is above 1), head_dim
 * contiguous. */
typedef struct cs_tensor {
    void *data;
    int64_t batch_stride, token_stride, head_stride;
} cs_tensor;

#define CS_MAX_HEAD_DIM 128
#define CS_MAX_ATTENTION_SCALE 1024.0f

typedef struct cs_attention_args {
    int32_t type;                 /* CS_TYPE_* of q, k, v, o and their gradients */
    int32_t batch, heads, kv_heads; /* heads is a multiple of kv_heads; head h reads kv head h / (heads / kv_heads) */
    int32_t head_dim;             /* a multiple of 8, at most CS_MAX_HEAD_DIM */
    int32_t q_len, kv_len;        /* tokens of q and o; of k and v (a cache's capacity) */
    int32_t window, sinks;
    float scale;                  /* finite, in [0, CS_MAX_ATTENTION_SCALE] */
    const int32_t *q_lens;        /* device, [batch]: queries of each sequence; NULL: q_len */
    const int32_t *kv_lens;       /* device, [batch]: keys of each sequence; NULL: kv_len */
    cs_tensor q, k, v, o;
    float *lse;                   /* [batch, heads, q_len] natural log-sum-exp; may be NULL in cs_attention */
} cs_attention_args;

/* o = softmax(scale q k^T) v. Scores are binary32 in units of log2: one of 2.3e38
 * and more in magnitude counts as infinite. The queries of a sequence are its last ones:
 * query i is at position kv_lens[b] - q_lens[b] + i. Lengths are clipped to
 * [0, q_len] and [0, kv_len]. Rows behind a sequence's queries are written as
 * rows that see no key; keys and values behind its length, and those that no
 * query sees, may hold anything. (A NaN or infinity in a value that some query
 * of the sequence sees may also reach other queries of that sequence that do
 * not see it.) A row whose visible scores are all -infinity is like one that
 * sees no key; one with a NaN or +infinity among them is NaN. One call serves
 * prompts, chunks of prompts over a cache (q_len < kv_len) and single tokens
 * (q_len 1). Probabilities are rounded to 16 bits before they meet the values, but
 * for few queries (up to 8, in some shapes 16, of a kv head's heads together),
 * where nothing is rounded but the result. `workspace`: at least
 * cs_attention_workspace bytes (0 for most shapes). */
int64_t cs_attention_workspace(const cs_attention_args *args);
int cs_attention(const cs_attention_args *args, void *workspace, size_t workspace_bytes, void *stream);

/* Gradients of q, k and v from that of o, with the o and lse that cs_attention
 * wrote for the same arguments. Rows of dq behind a sequence's queries, and
 * rows of dk and dv behind its keys, are written zero; what d_o holds there is
 * not used. Gradients of a kv head are summed over its query heads in binary32.
 * P and the gradient of the scores are rounded to 16 bits on the way. In fp16 the
 * latter is scaled to the largest that a row of dq, or the queries that see a tile of
 * 128 keys, can reach: smaller ones beside it are kept down to 2^-39 of that.
 * A NaN or infinity in a row of q, d_o or o, or in a key or value that is seen,
 * may reach all gradients of its sequence.
 * `workspace`: at least cs_attention_backward_workspace bytes. */
typedef struct cs_attention_grads {
    cs_tensor d_o, dq, dk, dv;
} cs_attention_grads;

int64_t cs_attention_backward_workspace(const cs_attention_args *args);
int cs_attention_backward(const cs_attention_args *args, const cs_attention_grads *grads,
                          void *workspace, size_t workspace_bytes, void *stream);

/* Every device-side wait of these kernels is bounded (2 s of GPU time); one
 * that runs out sets CS_STATUS_TIMEOUT in a status word of the current device.
 * Reads, then clears, that word: ordered on `stream`, which it waits for.
 * Returns cs_status_error of the bits. */
int cs_attention_status(uint32_t *status, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* CAUSAL_ATTENTION_H */
