/*
 * aps_decode.h -- C ABI of a decode step's operators around the paged cache of
 * aps_serve.h: rotary positions in the layouts and scalings of other models than
 * the reference's, linear layers with weights in 4 bits, and the log
 * probabilities of tokens.
 *
 * Same conventions as aps_moe.h (status codes, aps_moe_last_error, streams,
 * caller-owned device memory): every call is asynchronous on `stream`, on the
 * current device, allocates nothing and reads nothing back, so it can be
 * recorded into a HIP graph.  The reference has no counterpart: it rotates
 * halves of whole heads in fp32 (src/tensor.cu:2180-2197), keeps its weights in
 * fp32 and returns logits.
 */
#ifndef APS_DECODE_H
#define APS_DECODE_H

#include "aps_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rotary positions.  The first rotary_dim values of every head turn, pair i by
 * the angle positions[row] freq[i]:
 *   y0 = amplitude (x0 cos - x1 sin), y1 = amplitude (x0 sin + x1 cos),
 * the pairs being (i, i + rotary_dim / 2) (APS_ROPE_HALF, the layout of
 * aps_kv_append) or (2 i, 2 i + 1) (APS_ROPE_PAIRS); the rest of a head is
 * copied.  inverse: by the angle's negative (the transpose: the gradient, and
 * with amplitude 1 the way back).  freq [rotary_dim / 2] in 64 bits, as are the
 * angles; sines, products and sums are fp32, rounded once to the type.
 * q [rows][q_heads][head_dim] and k [rows][k_heads][head_dim] of dtype (F32 or
 * BF16) with row strides in elements, at any alignment of their elements (16-byte
 * accesses where all allow them); k NULL with k_heads 0: q alone.  A negative
 * position copies its row.  q_out may be q and k_out k with their strides;
 * outputs overlap nothing else of the call (refused).
 * rotary_dim is even, 2 .. head_dim; head_dim up to 1024. */
#define APS_ROPE_HALF 0
#define APS_ROPE_PAIRS 1
APS_API int aps_rope(const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, int32_t q_heads,
                     const void* k, int64_t k_stride, void* k_out, int64_t k_out_stride, int32_t k_heads,
                     int32_t dtype, int64_t rows, int32_t head_dim, int32_t rotary_dim, int32_t layout,
                     int32_t inverse, const int32_t* positions, const double* freq, float amplitude, void* stream);

/* The tables that aps_kv_append takes, from such frequencies: cos_table and
 * sin_table [count][pairs] of the positions first .. first + count - 1, times
 * amplitude. */
APS_API int aps_rope_freq_table(const double* freq, int32_t pairs, int64_t first, int64_t count, float amplitude,
                                float* cos_table, float* sin_table, void* stream);

/* A weight in 4 bits: w[n][k] = (code - zero) scale.  codes [out_features]
 * [in_features / 2], two to a byte, the even input in the low half, 16-byte
 * aligned; scales [out_features][in_features / group] of scale_dtype (F32 or
 * BF16); zeros [out_features][in_features / group] bytes, or NULL: 8.
 * group: 32, 64 or 128; in_features a multiple of it. */
typedef struct aps_q4_weight {
    const void* codes;
    const void* scales;
    const void* zeros;
    int32_t out_features;
    int32_t in_features;
    int32_t group;
    int32_t scale_dtype;
} aps_q4_weight;

/* y = x W^T + bias: x [rows][in_features] of dtype (F32 or BF16) with a row
 * stride in elements, bias [out_features] fp32 or NULL, y [rows][out_features]
 * contiguous of x's type.  Products are exact, sums are fp32, over each group's
 * codes and then over the groups; y is rounded once.  A row with an infinity or a
 * NaN gives NaN where the formula may have an infinity, and so may one with a
 * magnitude past 2^116, of which a group's sum need not be finite.  Of fp32 x the bits
 * below 2^-133, bf16's smallest number, are left out.  A scale that is
 * not finite makes its own output's values NaN or infinite, and no other's.  Any
 * alignment of x and y to their elements (16-byte reads where x allows them).
 * The kernel, and with it the order of the sums and the last bits of a row, goes by
 * the number of rows and the weight's sizes: a row alone and the same row in a batch
 * may differ by that rounding.  Equal calls give equal bits.
 * rows * in_features and rows * out_features up to 2^38.
 * workspace: aps_linear_q4_workspace_size bytes (0 for few rows), 16-byte aligned;
 * calls that overlap need one each.  y and workspace overlap nothing else of the call
 * (refused). */
APS_API size_t aps_linear_q4_workspace_size(const aps_q4_weight* weight, int64_t rows, int32_t dtype);
APS_API int aps_linear_q4(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, const aps_q4_weight* weight,
                          const float* bias, void* y, void* workspace, size_t workspace_bytes, void* stream);

/* Fills weight's arrays from w [out_features][in_features] (contiguous, F32 or
 * BF16, 16-byte aligned).  A group's scale, rounded to scale_dtype, is
 * max |w| / 7 without zeros; with them (max(w, 0) - min(w, 0)) / 15, and the zero
 * is min(w, 0) / -scale to nearest even, cut to 0 .. 15.  A scale of 0 is held
 * as 1.  Codes are w / scale to nearest even, plus the zero, cut to 0 .. 15.  A
 * group with an infinity or a NaN has the scale NaN. */
APS_API int aps_quantise_q4(const void* w, int32_t dtype, const aps_q4_weight* weight, void* stream);

/* Log probabilities under rows of logits [rows][vocab] (F32 or BF16, a row stride
 * in elements, any alignment of its elements), in fp32, all outputs fp32 and
 * contiguous:
 *   logprobs [rows][n_tokens]: logits[r][t] - log sum_j exp(logits[r][j]) of the
 *     given tokens [rows][n_tokens]; 0 for an id outside the vocabulary (padding)
 *   entropy [rows] (or NULL): -sum_j p_j log p_j
 *   top_ids, top_logprobs [rows][top]: the row's likeliest tokens, the likeliest
 *     first, of equal logits the lower id; a NaN counts as -inf.
 * Logits of -inf (a mask's) have the probability 0 and the log probability -inf;
 * a row of nothing else has these for all, and the entropy 0.  A row with NaN or
 * +inf gives NaN (but its top_ids).  Masks of -inf cost nothing; under one of a finite
 * value that leaves a row few tokens, as with many equal logits at the top, each of
 * the `top` tokens costs a pass over the row.  top up to 64 and vocab, vocab up to 2^20.
 * The order of the sums goes by rows, vocab, dtype and where a row begins within 16
 * bytes; equal calls on equally aligned rows give equal bits.
 * workspace: aps_token_logprobs_workspace_size bytes (0: none), 16-byte aligned;
 * calls that overlap need one each. */
APS_API size_t aps_token_logprobs_workspace_size(int64_t rows, int64_t vocab, int32_t top, int32_t dtype);
APS_API int aps_token_logprobs(const void* logits, int64_t logits_stride, int32_t dtype, int64_t rows, int64_t vocab,
                               const int32_t* tokens, int64_t n_tokens, int32_t top, float* logprobs, float* entropy,
                               int32_t* top_ids, float* top_logprobs, void* workspace, size_t workspace_bytes,
                               void* stream);

#ifdef __cplusplus
}
#endif

#endif /* APS_DECODE_H */
