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
// The most workgroups of a launch, bytes of `part`, and the launches; all follow
// one plan of the sizes.
int64_t attention_paged_blocks(const KvCache& cache, const PagedArgs& a);
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
