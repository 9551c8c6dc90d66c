/* ember_kv4.h — operators for decoding many streams: a paged KV cache held in 4
 * bits, attention over it, and one draw per row of a batch of logits.
 *
 * No counterpart in emberllm (one sequence per state, fp32 / fp16 cache, sampling
 * on the host). The operators work on device memory that the caller owns, allocate
 * nothing, run on the caller's stream and may be captured into a graph. They
 * return 0, or 1 with a message in ember_cuda_error(); nothing has been enqueued
 * then. The work runs on the device that owns the buffers; the caller's current
 * device is unchanged on return. Host arguments are checked on the host. Lengths
 * and page numbers live on the device: the kernels bound every index they form
 * from them (see each operator), so wrong ones give wrong results but touch no
 * memory outside the buffers.
 *
 * Only plain C types cross this boundary.
 */
#ifndef EMBER_B200_KV4_H
#define EMBER_B200_KV4_H

#include <stddef.h>
#include <stdint.h>

#include "ember.h"
#include "ember_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the cache ----
 * n_pages pages of page_size positions, each with the keys and values of every kv
 * head of one layer, in blocks of 32 consecutive elements with the values of
 * Q4_0: (code - 8) * d, codes 0..15, d an fp16 number. d is the block's first
 * value of largest magnitude divided by -8, rounded to 8 significant bits (as
 * bf16 does, to nearest even) and then to fp16, at most 8160 in magnitude; the
 * code of x is floor(x / d + 8.5) in exact arithmetic, clamped to 0..15 (8 where
 * d is 0). With so short a d every cached value is exactly an fp16 number. A NaN
 * is stored as 0 and an infinity as the largest value the block can hold: the
 * cache never holds either.
 *
 * The order of the bytes inside a page is the kernels' own: only the functions
 * below read or write it. Bytes never written may have any content: positions
 * that no row of a call sees (behind a sequence's length, in front of its rows' window)
 * have no part in the result. */
typedef struct {
    void   *data;         /* device memory of this layer's cache, 16-byte aligned     */
    int32_t n_pages;      /* n_pages * page_size at most 2^31 - 1                     */
    int32_t page_size;    /* 16, 32, 64 or 128                                        */
    int32_t n_kv_heads;
    int32_t head_dim;     /* 32, 64 or 128                                            */
} EmberKv4Cache;

/* bytes of `data` for such a cache; 0 when a number is not allowed */
size_t ember_cuda_kv4_bytes(int32_t n_pages, int32_t page_size, int32_t n_kv_heads, int32_t head_dim);

/* Which rows of a batch belong to which sequence and where its pages are. Sequence
 * i has kv_len[i] positions in the cache (the rows of this call included), and its
 * rows q_start[i] .. q_start[i+1]-1 are the last ones: row q_start[i+1]-1 is position
 * kv_len[i]-1. Position p lies in page block_table[i][p / page_size].
 * All three arrays are device memory. */
typedef struct {
    const int32_t *q_start;      /* [n_seqs + 1]; NULL: one row per sequence, row i          */
    const int32_t *kv_len;       /* [n_seqs]                                                 */
    const int32_t *block_table;  /* [n_seqs][table_stride]                                   */
    int32_t n_seqs;              /* at most 65535                                            */
    int32_t table_stride;
    int32_t n_tokens;            /* rows of the batch's tensors                              */
    int32_t max_q;               /* no sequence has more rows than this (1 when q_start NULL)*/
} EmberKv4Batch;

/* Quantize the rows' keys and values into the cache. k and v are [n_tokens]
 * [n_kv_heads][head_dim] of dtype EMBER_DT_F32 or EMBER_DT_F16, a head's elements
 * consecutive, *_tok and *_head the other strides in elements. Rows whose position
 * is negative or behind the table, or whose table entry is no page, are not stored.
 * One call must not store the same position of the same page twice. */
typedef struct {
    const void *k, *v;
    int32_t dtype;
    int64_t k_tok, k_head, v_tok, v_head;
} EmberKv4Rows;
int ember_cuda_kv4_store(const EmberKv4Cache *cache, const EmberKv4Batch *batch, const EmberKv4Rows *rows,
                         void *stream);

/* The inverse: the cached values of the rows' positions into k and v (which must
 * be writable). Rows that store would not have stored are left as they are. */
int ember_cuda_kv4_read(const EmberKv4Cache *cache, const EmberKv4Batch *batch, const EmberKv4Rows *rows,
                        void *stream);

/* Attention of the rows' queries over the cache: per row at position pos and per
 * query head, softmax over the visible positions p of scale * (q . k_p), times v_p.
 * Query head h reads kv head h / (n_heads / n_kv_heads). Visible are p <= pos with
 * a valid page and, when window > 0, only those with pos - p < window or
 * p < sinks (the first tokens that stay visible). A row that sees nothing gets
 * zeros. q and out are [n_tokens][n_heads][head_dim] of dtype F32 or F16; rows
 * that belong to no sequence are left as they are. A NaN or an infinity in a query
 * makes that (row, head)'s output NaN and no other.
 *
 * Arithmetic: the queries enter the products in 22 significant bits relative to
 * the row's largest element, the softmax weights in 22 bits; scores, maxima, sums
 * and outputs accumulate in fp32. Many-row calls (prompts) add on the tensor cores,
 * which cut toward zero: 2.5e-9 of an output a position, for fp32 over 512 positions
 * at most (1.6e-6 of an output at any length), for fp16 over all (1e-4 at 40,000).
 * They keep partial sums in `out` while they run. out may be q itself.
 * The same call gives the same bits. A row's result does not depend on its
 * neighbours in the batch; in the last bits it depends on how the cache is cut into
 * pieces, which follows from n_tokens, n_seqs, max_q, max_kv, window and sinks.
 *
 * max_kv bounds kv_len (positions behind it are not looked at). workspace: device
 * memory of at least ember_cuda_kv4_attention_workspace() bytes, 16-byte aligned,
 * contents irrelevant before and after; calls that overlap on the GPU (other
 * streams, graphs replayed at once) need one each. */
typedef struct {
    const void *q;
    void *out;
    int32_t dtype;
    int32_t n_heads;             /* a multiple of n_kv_heads                         */
    int64_t q_tok, q_head, out_tok, out_head;
    float scale;                 /* finite                                           */
    int32_t max_kv;
    int32_t window, sinks;       /* window 0: every position up to the row's own     */
    void *workspace;
    size_t workspace_bytes;
} EmberKv4Attention;
size_t ember_cuda_kv4_attention_workspace(const EmberKv4Cache *cache, int32_t n_heads, int32_t n_seqs, int32_t max_q,
                                          int32_t max_kv);
int ember_cuda_kv4_attention(const EmberKv4Cache *cache, const EmberKv4Batch *batch, const EmberKv4Attention *att,
                             void *stream);

/* Waits for the stream's work and returns 1 when a wait inside an attention call on the
 * cache's device has run out since this was last asked (a second of waiting, which no working
 * GPU needs): the rows it concerned are NaN. Not while the stream is captured. */
int ember_cuda_kv4_status(const EmberKv4Cache *cache, void *stream);

/* ---- one draw per row ----
 * out[r] = a token drawn from row r of logits [n_rows][vocab] (dtype F32 or F16, row
 * stride in elements, a row's elements consecutive), with that row's settings and
 * its own random number u[r] in [0, 1). The steps of ember_sample_device without the
 * penalties, in exact order instead of the reference's rounded one:
 *   order       logits descending, equal ones by index ascending; a NaN counts as -inf
 *   weight      w = exp((logit - max) / temperature)
 *   kept        the first top_k of the order (0 or less: all), of those the ones with
 *               w >= min_p (outside (0, 1): all), of those the shortest prefix whose
 *               weights reach top_p of the whole row's (outside (0, 1): all)
 *   draw        the first kept token whose running weight exceeds u * (kept weight);
 *               u outside [0, 1) counts as its nearest end, a NaN as 0
 * A temperature of 0 or less (or NaN) gives the first index of the maximum; so does a
 * row whose logits are all -inf or NaN (index 0). Weights are exp in double precision,
 * held as multiples of 2^-44 and added as integers: neither the order of the additions
 * nor the other rows can change a token. temperature, top_k, top_p, min_p and u are
 * device arrays of n_rows; NULL means 1, all, all, all (u is required). */
#define EMBER_SAMPLE_MAX_VOCAB 393216
typedef struct {
    const void *logits;
    int32_t dtype, n_rows, vocab;        /* vocab in [1, EMBER_SAMPLE_MAX_VOCAB] */
    int64_t stride;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *out;
} EmberSampleRows;
int ember_cuda_sample_rows(const EmberSampleRows *args, void *stream);

/* ---- streams over a paged 4-bit cache, and drawn steps ----
 * A batch of independent streams (ember_cuda_batch_*, ember_batch_*) whose caches are
 * pages of 64 positions in 4 bits, taken from one pool of n_pages (0: enough for every
 * stream's whole context) when a prompt or a step needs them. Keys and values are
 * quantized, so tokens may differ from those over an fp32 or fp16 cache; attention is
 * ember_cuda_kv4_attention's, with `window` and `sinks`. Any n_streams in [1, 512];
 * head_dim 32, 64 or 128. prefill, greedy, sample and free take such a batch as any
 * other. What other streams hold or do has no part in a stream's results; past 512
 * positions the last bits of its attention depend on n_streams, which decides how a cache
 * is cut into pieces.
 * A call that finds no free page fails and leaves the streams as they were
 * (pages handed out before it found out stay with their streams). Pages behind the
 * window stay, too.
 * release gives a stream's pages back and leaves it idle until its next prompt, which
 * starts anew: greedy and sample go on without it. Its toks, pos, params and u are not
 * looked at then, it takes no page, its tokens are -1 and its logits 0. */
int ember_cuda_batch_new_kv4(EmberCudaModel *m, int n_streams, int ctx, int n_pages, int window, int sinks,
                             const float *rope_cs, int max_steps, EmberCudaBatch **out);
int ember_cuda_batch_release(EmberCudaBatch *b, int stream);
int ember_cuda_batch_idle(const EmberCudaBatch *b, int stream);     /* 1 or 0 */
/* As ember_cuda_batch_greedy, but every step's tokens are drawn by
 * ember_cuda_sample_rows: stream i with params[i] (no penalties) and, at step t, the
 * random number u[t * n_streams + i]. Not for a batch that holds one state per stream
 * (up to 8 streams over an fp32 or fp16 cache). */
int ember_cuda_batch_sample(EmberCudaBatch *b, const int *toks, const int *pos, int n_steps,
                            const EmberSampleParams *params, const float *u, int *host_tokens, float *host_logits);

/* the same on the public batch; fatal errors follow the library's convention */
EmberBatch *ember_batch_new_kv4(EmberModel *m, int n_streams, int ctx_len, int n_pages, int window, int sinks,
                                int max_steps);
void ember_batch_release(EmberBatch *b, int stream);
void ember_batch_sample(EmberBatch *b, const int *toks, const int *pos, int n_steps, const EmberSampleParams *params,
                        const float *u, int *out_tokens, float *out_logits);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif /* EMBER_B200_KV4_H */
