/*
 * aps_serve.h -- C ABI of the serving operators: a paged key/value cache,
 * attention over it, and the rules on the logits of the next token.
 *
 * Same conventions as aps_moe.h (status codes, aps_moe_last_error, streams,
 * caller-owned device memory): every call is asynchronous on `stream`, on the
 * current device, allocates nothing and reads nothing back, so it can be
 * recorded into a HIP graph.  The reference has no counterpart: its
 * generate_decode computes the whole prefix again for every token
 * (src/model.cu:163-204).
 */
#ifndef APS_SERVE_H
#define APS_SERVE_H

#include "aps_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Cache element types: APS_DTYPE_F32, APS_DTYPE_BF16 and 4 bits. */
#define APS_KV_MXFP4 3

/* One layer's cache.  A page holds page_size consecutive positions of one
 * sequence, for every head; slot s is position s % page_size of page
 * s / page_size.  k and v are [num_pages][kv_heads][page_size][head_dim], 16-
 * byte aligned.  APS_KV_MXFP4 holds blocks of 32 values along head_dim as the
 * 4-bit floats e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign bit, two codes to a
 * byte, the even index in the low half: k, v [..][head_dim / 2] bytes) times
 * one power of two 2^(b - 127) a block (k_scale, v_scale [..][head_dim / 32]
 * bytes, 4-byte aligned): the smallest that keeps the block's largest
 * magnitude at 6 or below, so no value saturates.  A block with a NaN or an
 * infinity has b = 255 and reads back as NaN.
 * page_size: 16, 32, 64, 128 or 256; head_dim: 64 or 128; num_pages * page_size
 * up to 2^40. */
typedef struct aps_kv_cache {
    void* k;
    void* v;
    void* k_scale;      /* NULL unless MXFP4 */
    void* v_scale;
    int64_t num_pages;
    int32_t page_size;
    int32_t kv_heads;
    int32_t head_dim;
    int32_t dtype;
} aps_kv_cache;

/* Writes the keys and values of new tokens into the cache, the keys rotated
 * by their positions on the way, and rotates the queries:
 *   x0' = x0 c - x1 s, x1' = x0 s + x1 c for the pairs (j, j + head_dim / 2),
 * c, s = cos_table / sin_table [max_pos][head_dim / 2] at positions[row]
 * (aps_rope_table's), computed in 64 bits and rounded once to fp32, then to
 * the held type.  k, v [rows][kv_heads][head_dim] and q [rows][q_heads]
 * [head_dim] of src_dtype (F32 or BF16) with row strides in elements, so they
 * may be slices of one projection's rows.  q NULL: keys and values alone; else
 * q_out takes the rotated queries in src_dtype (q_out may be q itself with q's
 * stride; its rows overlap nothing else, refused for those of q, k and v and the
 * cached values).
 * Row r goes to slots[r]; a slot outside the cache (-1: padding) writes no key
 * and no value.  Slots of one call are distinct: of rows that name the same
 * slot either may stay, element by element.  A position outside [0, max_pos)
 * leaves its row unrotated.  An F32 cache takes F32 sources.
 * Any 4-byte (BF16: 2-byte) alignment; 16-byte accesses where sources, tables,
 * q_out and strides allow them. */
APS_API int aps_kv_append(const aps_kv_cache* cache, const void* k, int64_t k_stride, const void* v,
                          int64_t v_stride, const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride,
                          int32_t src_dtype, int64_t rows, int32_t q_heads, const int32_t* positions,
                          const int64_t* slots, const float* cos_table, const float* sin_table, int64_t max_pos,
                          void* stream);

/* Reads cached rows back: k_out, v_out [rows][kv_heads][head_dim] of out_dtype
 * (F32, or BF16 rounded to nearest even; 16-byte aligned), the values that the
 * codes of a 4-bit cache stand for.  Either may be NULL.  A slot outside the
 * cache gives a row of zeros.  The outputs overlap nothing else (refused for each
 * other and the cached values). */
APS_API int aps_kv_gather(const aps_kv_cache* cache, const int64_t* slots, int64_t rows, void* k_out, void* v_out,
                          int32_t out_dtype, void* stream);

/* Softmax attention of each sequence's newest tokens over its cached keys.
 * Sequence b has kv_lens[b] cached positions, its new tokens among them:
 * position j is at offset j % page_size of page page_table[b][j / page_size].
 * Its queries are rows q_offsets[b] .. q_offsets[b + 1] - 1 of q [rows]
 * [q_heads][head_dim] (row stride q_stride elements), the last of them at
 * position kv_lens[b] - 1.  The query at position p sees the keys j <= p with
 * j > p - window or j < sinks: a sliding window and the first tokens.
 *   out = sum_j exp(scale q.k_j) v_j / sum_j exp(scale q.k_j), out [rows]
 * [q_heads][head_dim] contiguous, of q's type.  q_heads is a multiple of
 * kv_heads; query head h reads key head h / (q_heads / kv_heads).  scale log2 e
 * has to be finite in fp32.
 * q_dtype F32 takes every cache type, BF16 the BF16 and MXFP4 ones.  Products
 * are exact and sums are fp32; with BF16 queries the softmax weights are held
 * for their product with v to 16 bits, and of a sequence with more than 32 rows
 * (tokens times q_heads / kv_heads) to bf16's 8.  (Shorter sequences beside
 * padding rows share the 8 where max_q_len is past 32 rows and rows >
 * (batch - 1) max_q_len + 32 / (q_heads / kv_heads): no room but for padding.)
 *
 * All arrays in device memory; q_offsets ascend; batch up to 2^20, max_kv_len up
 * to 2^30 (sizes that take 2^32 threads and more in a launch are refused).  max_q_len
 * and max_kv_len bound the batch's lengths on the host (they shape the launch, so a
 * recorded graph serves any lengths within them): queries past max_q_len of a
 * sequence are left as they were, lengths past max_kv_len or past table_stride
 * pages are cut.
 * Rows of out that no sequence names are left as they were.  A query that sees
 * no key (kv_lens[b] below its queries' number, or 0), or whose every score is
 * -inf, gives zeros.  A page id outside the cache leaves its keys out; entries
 * for pages that no query sees may hold anything.  Values and keys that a row does
 * not see do not reach it, infinities and NaN among them; of those that it does
 * see, NaN may stand where the formula has an infinity.
 * workspace: aps_attention_paged_workspace_size bytes (0: none), 256-byte
 * aligned; calls that overlap need one each.  q, out 16-byte aligned, q_stride
 * a multiple of 16 bytes.  out and workspace overlap nothing else of the call
 * (refused for q, out and workspace). */
APS_API size_t aps_attention_paged_workspace_size(const aps_kv_cache* cache, int64_t rows, int32_t q_heads,
                                                  int64_t batch, int64_t max_q_len, int64_t max_kv_len,
                                                  int32_t window, int32_t sinks);
APS_API int aps_attention_paged(const aps_kv_cache* cache, const void* q, int64_t q_stride, int32_t q_dtype,
                                int64_t rows, int32_t q_heads, const int32_t* q_offsets, const int32_t* kv_lens,
                                const int32_t* page_table, int64_t table_stride, int64_t batch, int64_t max_q_len,
                                int64_t max_kv_len, int32_t window, int32_t sinks, float scale, void* out,
                                void* workspace, size_t workspace_bytes, void* stream);

/* The rules between the LM head and the choice of a token.  Every array is
 * device memory and a NULL one is a rule that is off.
 * history [rows][history_stride]: the token ids of each row so far, the first
 * history_lens[r] of them (ids outside the vocabulary count for nothing); the
 * first prompt_lens[r] are its prompt (NULL: none of them). */
typedef struct aps_logits_rules {
    const int32_t* history;
    const int32_t* history_lens;
    const int32_t* prompt_lens;
    int64_t history_stride;
    const float* repetition;   /* [rows], > 0 */
    const float* frequency;    /* [rows] */
    const float* presence;     /* [rows] */
    const int32_t* bias_ids;   /* [rows][bias_stride], the first bias_lens[r] */
    const float* bias_values;  /* [rows][bias_stride]; of an id named twice the last value counts */
    const int32_t* bias_lens;
    int64_t bias_stride;
    const uint32_t* mask;      /* [mask_rows][mask_stride words]: bit t % 32 of word t / 32 allows token t */
    int64_t mask_rows;
    int64_t mask_stride;
    const int32_t* mask_index; /* [rows]: the row's mask; outside [0, mask_rows): none.  NULL: row r has mask r */
} aps_logits_rules;

/* out[r][t] from x = logits[r][t] (F32 or BF16, row strides in elements; out
 * may be logits itself with its stride, and overlaps nothing else of the call:
 * other rows over logits' are refused), in fp32, rounded once:
 *   t anywhere in the history:     x = x > 0 ? x / repetition : x * repetition
 *   t n > 0 times past the prompt: x = x - frequency n, then x - presence
 *   t in the bias list:            x = x + its value
 *   t not allowed by the mask:     x = -inf
 * Columns past vocab of a wider row are left as they were. */
APS_API int aps_logits_process(const void* logits, int64_t logits_stride, int32_t dtype, int64_t rows, int64_t vocab,
                               const aps_logits_rules* rules, void* out, int64_t out_stride, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* APS_SERVE_H */
