/*
 * qgops.h -- C ABI of the operators around the mat-vecs of libqgemv: a KV
 * cache held in 8 bits, attention over it, and the log probabilities of
 * tokens.
 *
 * yudono/rust-inference keeps one f32 cache per layer for one sequence
 * (KVCache, src/kv_cache.rs:40-90), attends over it one token at a time
 * (Attention::forward, src/attention.rs:89-121) and answers with a sampled
 * token (src/sampler.rs:72-83).  These operators have no counterpart there:
 * the cache takes a quarter of the bytes, holds several sequences, takes whole
 * prompts and single tokens in one call, and the logits also answer with
 * probabilities.  qg_model_use_kv8 and qg_model_logprobs (qgmodel.h) use them
 * in the decode step's model.
 *
 * Status codes are qg_status values (qgemv.h).  Every `_dev` call takes device
 * pointers, is asynchronous on `stream` (a hipStream_t, NULL = the context's
 * own stream), allocates nothing, waits for nothing and can be captured into a
 * HIP graph: what changes from step to step (the cached positions, the rows of
 * each sequence) is read from device memory when the kernels run.
 */
#ifndef QGOPS_H
#define QGOPS_H

#include <stddef.h>
#include <stdint.h>

#include "qgemv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows of a batch, [row][head][head_dim] on the device: element d of head h of
 * row r at data[r * ld_row + h * ld_head + d] (strides in elements, so q, k and
 * v may be parts of one buffer, and heads may come before rows).  type: the
 * GGML id of f32 (0) or f16 (1); any other: QG_ERR_UNSUPPORTED_TYPE.  data is
 * aligned to its element; rows that are also aligned to 16 bytes, with a
 * head_dim of whole 16 elements, are read and written fastest.  Written rows
 * must not overlap one another (QG_ERR_SHAPE) nor anything that the same call
 * reads. */
typedef struct qg_rows {
    void *data;
    uint32_t type;
    size_t ld_row, ld_head;
} qg_rows;

/* Which rows of a call belong to which sequence of the cache, and where they
 * stand.  Sequence s has the rows d_starts[s] .. d_starts[s + 1) (n_seqs + 1
 * values, not decreasing, the last one at most n_rows), or, with d_starts
 * NULL, the single row s (n_rows must then be n_seqs, else QG_ERR_SHAPE).
 * n_rows is below 2^28 (QG_ERR_SHAPE).
 * d_lens[s] counts its positions with this call's tokens included: row i of
 * its n rows stands at position d_lens[s] - n + i.  A sequence without rows
 * takes no part; rows behind the last sequence's are neither read nor
 * written; a row at a position below 0 or not below max_len is not cached.
 * Both arrays are device memory, read when the kernels run. */
typedef struct qg_batch {
    size_t n_rows;
    const uint32_t *d_starts;
    const uint32_t *d_lens;
} qg_batch;

/* The keys and values of one attention layer for n_seqs sequences of up to
 * max_len positions.  Positions are held in blocks of QG_KV8_BLOCK; the values
 * x of a block and head are codes in -127 .. 127 under one f32 scale,
 *   scale = max |x| / 127 (zero where that is below 2^-126),
 *   code = x / scale to the nearest, ties to even,   x ~ code * scale,
 * over the positions written so far.  A block that is not full keeps its f32
 * values beside the codes, so a larger value in a later call has the block
 * quantised again from the values and not from codes: the cache depends on the
 * tokens alone, not on how they came in calls.  A block (of one head, keys or
 * values) that holds an infinity or a NaN reads as NaN, others are unaffected. */
typedef struct qg_kv8 qg_kv8;
enum { QG_KV8_BLOCK = 32 };

/* n_seqs, n_kv_heads 1 .. 65535 and 2^26 at most together, head_dim 1 .. 256,
 * max_len 1 .. 2^31 - 32 (QG_ERR_SHAPE otherwise).  An empty cache, all zero; synchronous. */
int qg_kv8_create(qg_ctx *ctx, size_t n_seqs, size_t n_kv_heads, size_t head_dim, size_t max_len, qg_kv8 **out);
/* QG_ERR_INVALID_ARG for a handle this context does not hold.  The caller has
 * waited for its own streams; qg_destroy frees what is left. */
int qg_kv8_free(qg_ctx *ctx, qg_kv8 *kv);
/* Any output may be NULL.  bytes: device memory of the cache. */
int qg_kv8_info(const qg_kv8 *kv, size_t *n_seqs, size_t *n_kv_heads, size_t *head_dim, size_t *max_len,
                size_t *bytes);

/* Caches k and v (n_kv_heads heads, the same type) of the batch's rows.
 * A sequence's tokens come in order: the positions before the call's have been
 * written.  Positions may be written again, and a sequence may go back: its
 * tokens from the call's first position on are the new ones.  Back inside the
 * block that was open before the last call, or the one open now, nothing is
 * lost; further back the earlier positions of a reopened block go on with
 * their 8-bit values.  Calls on one cache must not overlap. */
int qg_kv8_write_dev(qg_ctx *ctx, qg_kv8 *kv, const qg_batch *batch, const qg_rows *k, const qg_rows *v, void *stream);

/* Positions pos .. pos + n of sequences seq .. seq + n_seqs as values: row
 * (i * n + j) of k and v is position pos + j of sequence seq + i.  Either
 * output may be NULL.  QG_ERR_SHAPE outside the cache, for n of 2^28 or more, and
 * for keys and values of more than 65535 heads together.  Positions behind a
 * sequence's last read as zero in a new cache, else as what is left there. */
int qg_kv8_read_dev(qg_ctx *ctx, const qg_kv8 *kv, size_t seq, size_t n_seqs, size_t pos, size_t n, const qg_rows *k,
                    const qg_rows *v, void *stream);

/* Causal attention of the batch's rows (n_heads query heads, a multiple of
 * n_kv_heads: query head h reads kv head h / (n_heads / n_kv_heads)) over the
 * cached values, this call's tokens' among them (qg_kv8_write_dev first):
 *   out = sum_j p_j v_j,  p = softmax over j of scale * q . k_j,
 * for the row at position p over the positions j <= p, and j > p - window
 * where window is not 0.  Rows see the values as they are after the call's
 * writes: a later token of the same block may have moved its scale.  A row with
 * no position to see (one below 0) gives zeros; a row at a position past max_len
 * sees the positions there are.  n_heads at most 65535, n_rows * n_heads below
 * 2^31 (QG_ERR_SHAPE).  q and out have one type; f32 rows are computed to f32
 * precision (two f16 pieces of q and of p), f16 rows with f16 p, sums in f32.
 * d_work: qg_kv8_attention_work bytes of device memory (16-byte aligned) that no
 * other call in flight uses (captured graphs that may run side by side need one
 * each); its contents need not be kept.  QG_ERR_SHAPE when work_bytes is less. */
int qg_kv8_attention_dev(qg_ctx *ctx, const qg_kv8 *kv, const qg_batch *batch, size_t n_heads, const qg_rows *q,
                         float scale, size_t window, const qg_rows *out, void *d_work, size_t work_bytes,
                         void *stream);
/* Bytes of workspace a call with up to n_rows rows needs (may be 0). */
int qg_kv8_attention_work(qg_ctx *ctx, const qg_kv8 *kv, size_t n_rows, size_t n_heads, size_t *bytes);

/* For each of n_rows rows of n_cols logits x (type f32 or f16, ld elements
 * between rows): the log probability of n_given given tokens,
 *   lp(t) = x_t - m - log Z,  m = max x,  Z = sum exp(x - m),
 * into d_logprobs[row][n_given] (NULL with n_given 0; d_tokens[row][n_given]
 * token ids: QG_TOKEN_NONE gives 0, any other id >= n_cols NaN); the entropy
 * -sum p log p into d_entropy[row] (NULL: not wanted); and the k <= 64 most
 * likely tokens (k 0: none) into d_top_ids and d_top_logprobs[row][k], by
 * logit, equal ones by id.  A logit of -inf has probability 0.  A NaN is never
 * among the alternatives; places behind the row's tokens hold QG_TOKEN_NONE and
 * -inf.  In a row that holds a NaN or +inf, or -inf only, every probability and
 * the entropy are NaN (the ids still are the largest logits).  Sums in f32.
 * d_work: qg_logprobs_work bytes (16-byte aligned), as for
 * qg_kv8_attention_dev.  n_rows below 2^24, n_cols 1 .. 2^31 - 1, rows ld >=
 * n_cols apart (QG_ERR_SHAPE otherwise). */
enum { QG_LOGPROBS_MAX_TOP = 64 };
#define QG_TOKEN_NONE 0xFFFFFFFFu
int qg_logprobs_dev(qg_ctx *ctx, const void *d_logits, uint32_t type, size_t n_rows, size_t n_cols, size_t ld,
                    const uint32_t *d_tokens, size_t n_given, float *d_logprobs, float *d_entropy, size_t k,
                    uint32_t *d_top_ids, float *d_top_logprobs, void *d_work, size_t work_bytes, void *stream);
/* Bytes of workspace such a call needs (may be 0). */
int qg_logprobs_work(qg_ctx *ctx, size_t n_rows, size_t n_cols, size_t k, size_t *bytes);

#ifdef __cplusplus
}
#endif

#endif /* QGOPS_H */
