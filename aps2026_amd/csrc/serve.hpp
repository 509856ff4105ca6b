// Internal declarations of the serving operators: the paged cache, attention
// over it and the rules on logits.
#pragma once

#include "common.hpp"

namespace aps {

enum class Kv { kF32 = 0, kBf16 = 1, kMx = 3 };

struct KvCache {
    void *k, *v;
    uint8_t *k_scale, *v_scale;
    int64_t num_pages;
    int page_shift;  // log2 of the page size
    int kv_heads, head_dim;
    Kv type;
};

struct KvAppendArgs {
    const void *k, *v, *q;
    void* q_out;
    int64_t k_stride, v_stride, q_stride, q_out_stride;
    int64_t rows;
    int q_heads;  // 0 without q
    const int32_t* positions;
    const int64_t* slots;
    const float *cosv, *sinv;
    int64_t max_pos;
};
hipError_t launch_kv_append(const KvCache& cache, const KvAppendArgs& a, bool src_f32, hipStream_t s);
hipError_t launch_kv_gather(const KvCache& cache, const int64_t* slots, int64_t rows, void* k_out, void* v_out,
                            bool out_f32, hipStream_t s);

constexpr float kLog2e = 1.4426950408889634f;
struct PagedArgs {
    const void* q;
    int64_t q_stride;
    int64_t rows;
    int q_heads;
    const int32_t *q_offsets, *kv_lens, *page_table;
    int64_t table_stride, batch, max_q_len, max_kv_len;
    int window, sinks;
    float scale;
    void* out;
    float* part;  // partial results of a split key axis
};
// The most threads of a launch, bytes of `part`, and the launches; all follow
// one plan of the sizes.
int64_t attention_paged_threads(const KvCache& cache, const PagedArgs& a);
size_t attention_paged_part_bytes(const KvCache& cache, const PagedArgs& a);
hipError_t launch_attention_paged(const KvCache& cache, const PagedArgs& a, bool q_f32, hipStream_t s);

struct LogitsArgs {
    const void* x;
    void* out;
    int64_t x_stride, out_stride, rows, vocab;
    const int32_t *history, *history_lens, *prompt_lens;
    int64_t history_stride;
    const float *repetition, *frequency, *presence;
    const int32_t* bias_ids;
    const float* bias_values;
    const int32_t* bias_lens;
    int64_t bias_stride;
    const uint32_t* mask;
    int64_t mask_rows, mask_stride;
    const int32_t* mask_index;
};
hipError_t launch_logits_process(const LogitsArgs& a, bool f32, hipStream_t s);

struct RopeArgs {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_stride, q_out_stride, k_stride, k_out_stride;
    int64_t rows;
    int q_heads, k_heads;  // 0 without
    int head_dim, rotary_dim;
    bool pairs, inverse;
    const int32_t* positions;
    const double* freq;
    float amplitude;
};
hipError_t launch_rope(const RopeArgs& a, bool f32, hipStream_t s);
hipError_t launch_rope_table(const double* freq, int pairs, int64_t first, int64_t count, float amplitude,
                             float* cosv, float* sinv, hipStream_t s);

struct LogprobArgs {
    const void* x;
    int64_t x_stride, rows, vocab;
    const int32_t* tokens;
    int64_t n_tokens;
    int top;
    float *logprobs, *entropy;  // entropy may be null
    int32_t* top_ids;
    float* top_logprobs;
    float* part;  // a split row's parts
};
constexpr int kLogprobTop = 64;
constexpr int64_t kLogprobVocab = int64_t(1) << 20;
int64_t token_logprobs_blocks(int64_t rows, int64_t vocab, bool f32);
size_t token_logprobs_part_bytes(int64_t rows, int64_t vocab, int top, bool f32);
hipError_t launch_token_logprobs(const LogprobArgs& a, bool f32, hipStream_t s);

// Weights in 4 bits: w[n][k] = (code - zero) scale, a scale and a zero for each
// `group` neighbouring k.
struct Q4 {
    const uint8_t* codes;
    const void* scales;
    const uint8_t* zeros;  // null: 8
    int out, in, group;
    bool scales_f32;
};
struct LinearQ4Args {
    Q4 w;
    const void* x;
    int64_t x_stride, rows;
    const float* bias;
    void* y;          // [rows][out]
    uint16_t* terms;  // x in the products' order, for many rows
};
size_t linear_q4_bytes(const Q4& w, int64_t rows, bool f32);
hipError_t launch_linear_q4(const LinearQ4Args& a, bool f32, hipStream_t s);
hipError_t launch_quantise_q4(const void* w, bool w_f32, int64_t out, int in, int group, uint8_t* codes,
                              void* scales, bool scales_f32, uint8_t* zeros, hipStream_t s);

// ---- 4-bit blocks ----------------------------------------------------------

// The scale byte of a block from the largest |value| bits in it: with amax =
// 1.f 2^x the smallest e with amax <= 6 2^e = 1.5 2^(e + 2) is x - 2, or x - 1
// past 1.5; 1 (2^-126) at the least, 255 for an infinity or a NaN.
__device__ inline uint32_t mx_scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return 255u;
    const int b = static_cast<int>(amax_bits >> 23) - 2 + ((amax_bits & 0x7FFFFFu) > 0x400000u);
    return static_cast<uint32_t>(b < 1 ? 1 : b);
}
// The scale as the conversions take it (they read its exponent; 255 gives NaN).
__device__ inline float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Codes of 8 values, e2m1 of v / scale to nearest even (v_cvt_scalef32_pk_fp4_f32).
__device__ inline uint32_t mx_encode8(const float (&v)[8], float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
    return w;
}
// Two values of byte B of a word of codes as packed bf16: exact, a code has
// two significant bits.
template <int B>
__device__ inline uint32_t mx_decode2(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}

}  // namespace aps
