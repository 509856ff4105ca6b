// C ABI of a decode step's operators around the paged cache (declared in
// include/aps_decode.h): argument checks, then the launches.
#include "../../include/aps_decode.h"
#include "capi_args.hpp"
#include "serve.hpp"

namespace {

using namespace aps::args;
using aps::fail;

int check_dtype(int32_t dtype, const char* what) {
    if (dtype == APS_DTYPE_F32 || dtype == APS_DTYPE_BF16) return APS_OK;
    return fail(APS_ERR_DTYPE, "%s: dtype %d", what, dtype);
}

// A 4-bit weight's description; with `arrays` its pointers too.
int check_q4(const aps_q4_weight* d, const char* what, bool arrays, aps::Q4* out) {
    if (!d) return fail(APS_ERR_ARG, "%s: NULL weight", what);
    if (int rc = check_dtype(d->scale_dtype, what)) return rc;
    if (d->group != 32 && d->group != 64 && d->group != 128)
        return fail(APS_ERR_SHAPE, "%s: groups of %d (32, 64 or 128)", what, d->group);
    if (d->out_features < 1 || d->in_features < 1 || d->in_features % d->group != 0 || d->out_features > 1 << 24 ||
        d->in_features > 1 << 24)
        return fail(APS_ERR_SHAPE, "%s: a weight of %d x %d in groups of %d", what, d->out_features, d->in_features,
                    d->group);
    const uintptr_t elt = d->scale_dtype == APS_DTYPE_F32 ? 4 : 2;
    if (arrays) {
        if (!d->codes || !d->scales) return fail(APS_ERR_ARG, "%s: NULL weight array", what);
        if (mis(d->codes, 16) || mis(d->scales, elt))
            return fail(APS_ERR_ARG, "%s: codes must be 16-byte aligned, scales to their elements", what);
    }
    out->codes = static_cast<const uint8_t*>(d->codes);
    out->scales = d->scales;
    out->zeros = static_cast<const uint8_t*>(d->zeros);
    out->out = d->out_features;
    out->in = d->in_features;
    out->group = d->group;
    out->scales_f32 = d->scale_dtype == APS_DTYPE_F32;
    return APS_OK;
}
struct Q4Bytes {
    size_t codes, scales, zeros;
};
Q4Bytes q4_bytes(const aps::Q4& w) {
    const size_t n = static_cast<size_t>(w.out), groups = static_cast<size_t>(w.in / w.group);
    return {n * w.in / 2, n * groups * (w.scales_f32 ? 4 : 2), w.zeros ? n * groups : 0};
}
bool overlap_q4(const void* p, size_t np, const aps::Q4& w) {
    const Q4Bytes b = q4_bytes(w);
    return overlap(p, np, w.codes, b.codes) || overlap(p, np, w.scales, b.scales) ||
           overlap(p, np, w.zeros, b.zeros);
}

int check_linear_q4(const aps::Q4& w, int64_t rows, const char* what) {
    const int64_t wide = w.in > w.out ? w.in : w.out;
    if (rows < 0 || rows > kMaxRows || rows * wide > int64_t(1) << 38)
        return fail(APS_ERR_SHAPE, "%s: %lld rows of %d and %d values", what, (long long)rows, w.in, w.out);
    return APS_OK;
}

int check_logprobs(int64_t rows, int64_t vocab, int32_t top, int32_t dtype, const char* what) {
    if (int rc = check_dtype(dtype, what)) return rc;
    if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > aps::kLogprobVocab)
        return fail(APS_ERR_SHAPE, "%s: rows %lld, vocab %lld", what, (long long)rows, (long long)vocab);
    if (top < 0 || top > aps::kLogprobTop || top > vocab)
        return fail(APS_ERR_SHAPE, "%s: top %d of %lld (up to %d)", what, top, (long long)vocab, aps::kLogprobTop);
    if (aps::token_logprobs_blocks(rows, vocab, dtype == APS_DTYPE_F32) > 0x7FFFFFFF)
        return fail(APS_ERR_SHAPE, "%s: %lld rows of %lld logits", what, (long long)rows, (long long)vocab);
    return APS_OK;
}

}  // namespace

extern "C" {

int aps_rope(const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, int32_t q_heads, const void* k,
             int64_t k_stride, void* k_out, int64_t k_out_stride, int32_t k_heads, int32_t dtype, int64_t rows,
             int32_t head_dim, int32_t rotary_dim, int32_t layout, int32_t inverse, const int32_t* positions,
             const double* freq, float amplitude, void* stream) {
    const char* what = "rope";
    if (int rc = check_dtype(dtype, what)) return rc;
    if (head_dim < 2 || head_dim > 1024 || rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2 != 0)
        return fail(APS_ERR_SHAPE, "%s: %d rotary values of heads of %d", what, rotary_dim, head_dim);
    if (layout != APS_ROPE_HALF && layout != APS_ROPE_PAIRS) return fail(APS_ERR_ARG, "%s: layout %d", what, layout);
    if (rows < 0 || rows > kMaxRows || q_heads < 1 || q_heads > 65536 || k_heads < 0 || k_heads > 65536)
        return fail(APS_ERR_SHAPE, "%s: rows %lld, %d and %d heads", what, (long long)rows, q_heads, k_heads);
    const int64_t qd = static_cast<int64_t>(q_heads) * head_dim, kd = static_cast<int64_t>(k_heads) * head_dim;
    if (q_stride < qd || q_out_stride < qd || k_stride < kd || k_out_stride < kd)
        return fail(APS_ERR_SHAPE, "%s: row strides %lld, %lld of %lld values, %lld, %lld of %lld", what,
                    (long long)q_stride, (long long)q_out_stride, (long long)qd, (long long)k_stride,
                    (long long)k_out_stride, (long long)kd);
    if (!(amplitude - amplitude == 0.0f)) return fail(APS_ERR_ARG, "%s: amplitude is not finite", what);
    if ((q == q_out && q_stride != q_out_stride) || (k_heads && k == k_out && k_stride != k_out_stride))
        return fail(APS_ERR_ARG, "%s: rows turned in place keep their stride", what);
    if (rows == 0) return APS_OK;
    if (!q || !q_out || (k_heads && (!k || !k_out)) || !positions || !freq)
        return fail(APS_ERR_ARG, "%s: NULL pointer", what);
    const uintptr_t elt = dtype == APS_DTYPE_F32 ? 4 : 2;
    if (!k_heads) k = k_out = nullptr;
    if (mis(q, elt) || mis(q_out, elt) || mis(k, elt) || mis(k_out, elt) || mis(positions, 4) || mis(freq, 8))
        return fail(APS_ERR_ARG, "%s: arrays must be aligned to their elements", what);
    // a row is read after others were written
    const Rows from[2] = {rows_of(q, rows, qd, q_stride, elt), rows_of(k, rows, kd, k_stride, elt)};
    const Rows to[2] = {rows_of(q_out, rows, qd, q_out_stride, elt), rows_of(k_out, rows, kd, k_out_stride, elt)};
    for (int i = 0; i < 2; ++i)
        if ((from[i].at != to[i].at && overlap(to[i], from[i])) || overlap(to[i], from[1 - i]) ||
            overlap(to[i], {positions, 1, 4 * rows, 4 * rows}) ||
            overlap(to[i], {freq, 1, int64_t(4) * rotary_dim, int64_t(4) * rotary_dim}))
            return fail(APS_ERR_ARG, "%s: an output overlaps another array", what);
    if (overlap(to[0], to[1])) return fail(APS_ERR_ARG, "%s: q_out and k_out overlap", what);
    const aps::RopeArgs a{q,       k,        q_out,      k_out,  q_stride,                 q_out_stride, k_stride,
                          k_out_stride, rows, q_heads, k_heads, head_dim, rotary_dim, layout == APS_ROPE_PAIRS,
                          inverse != 0, positions, freq, amplitude};
    return launched(aps::launch_rope(a, dtype == APS_DTYPE_F32, static_cast<hipStream_t>(stream)), "rope launch");
}

int aps_rope_freq_table(const double* freq, int32_t pairs, int64_t first, int64_t count, float amplitude,
                        float* cos_table, float* sin_table, void* stream) {
    const char* what = "rope_freq_table";
    if (pairs < 1 || pairs > 512 || first < 0 || count < 0 || first > kMaxRows || count > kMaxRows ||
        first + count > kMaxRows || count * pairs > int64_t(1) << 38)
        return fail(APS_ERR_SHAPE, "%s: %d pairs at %lld positions from %lld", what, pairs, (long long)count,
                    (long long)first);
    if (!(amplitude - amplitude == 0.0f)) return fail(APS_ERR_ARG, "%s: amplitude is not finite", what);
    if (count == 0) return APS_OK;
    if (!freq || !cos_table || !sin_table) return fail(APS_ERR_ARG, "%s: NULL pointer", what);
    if (mis(freq, 8) || mis(cos_table, 4) || mis(sin_table, 4))
        return fail(APS_ERR_ARG, "%s: arrays must be aligned to their elements", what);
    const size_t bytes = static_cast<size_t>(count) * pairs * 4, from = static_cast<size_t>(pairs) * 8;
    if (overlap(cos_table, bytes, sin_table, bytes) || overlap(cos_table, bytes, freq, from) ||
        overlap(sin_table, bytes, freq, from))
        return fail(APS_ERR_ARG, "%s: a table overlaps another array", what);
    return launched(aps::launch_rope_table(freq, pairs, first, count, amplitude, cos_table, sin_table,
                                           static_cast<hipStream_t>(stream)),
                    "rope_freq_table launch");
}

size_t aps_linear_q4_workspace_size(const aps_q4_weight* weight, int64_t rows, int32_t dtype) {
    aps::Q4 w;
    if (check_q4(weight, "linear_q4", false, &w) || check_dtype(dtype, "linear_q4") ||
        check_linear_q4(w, rows, "linear_q4"))
        return 0;
    return aps::linear_q4_bytes(w, rows, dtype == APS_DTYPE_F32);
}

int aps_linear_q4(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, const aps_q4_weight* weight,
                  const float* bias, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "linear_q4";
    aps::Q4 w;
    if (int rc = check_q4(weight, what, rows > 0, &w)) return rc;
    if (int rc = check_dtype(dtype, what)) return rc;
    if (int rc = check_linear_q4(w, rows, what)) return rc;
    if (x_stride < w.in)
        return fail(APS_ERR_SHAPE, "%s: row stride %lld of %d values", what, (long long)x_stride, w.in);
    if (rows == 0) return APS_OK;
    if (!x || !y) return fail(APS_ERR_ARG, "%s: NULL pointer", what);
    const uintptr_t elt = dtype == APS_DTYPE_F32 ? 4 : 2;
    if (mis(x, elt) || mis(y, elt) || mis(bias, 4))
        return fail(APS_ERR_ARG, "%s: arrays must be aligned to their elements", what);
    const size_t need = aps::linear_q4_bytes(w, rows, dtype == APS_DTYPE_F32);
    if (need && (!workspace || workspace_bytes < need))
        return fail(APS_ERR_WORKSPACE, "%s: workspace %zu bytes, need %zu", what, workspace_bytes, need);
    if (need && mis(workspace, 16)) return fail(APS_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", what);
    const size_t out_bytes = static_cast<size_t>(rows) * w.out * elt, bias_bytes = static_cast<size_t>(w.out) * 4;
    const Rows from = rows_of(x, rows, w.in, x_stride, elt);
    const int64_t out_span = static_cast<int64_t>(out_bytes), ws_span = static_cast<int64_t>(need);
    if (overlap(Rows{y, 1, out_span, out_span}, from) || overlap(Rows{workspace, 1, ws_span, ws_span}, from) ||
        overlap(y, out_bytes, bias, bias ? bias_bytes : 0) || overlap(workspace, need, bias, bias ? bias_bytes : 0) ||
        overlap(y, out_bytes, workspace, need) || overlap_q4(y, out_bytes, w) || overlap_q4(workspace, need, w))
        return fail(APS_ERR_ARG, "%s: y or the workspace overlaps another array", what);
    const aps::LinearQ4Args a{w, x, x_stride, rows, bias, y, need ? static_cast<uint16_t*>(workspace) : nullptr};
    return launched(aps::launch_linear_q4(a, dtype == APS_DTYPE_F32, static_cast<hipStream_t>(stream)),
                    "linear_q4 launch");
}

int aps_quantise_q4(const void* w, int32_t dtype, const aps_q4_weight* weight, void* stream) {
    const char* what = "quantise_q4";
    aps::Q4 to;
    if (int rc = check_q4(weight, what, true, &to)) return rc;
    if (int rc = check_dtype(dtype, what)) return rc;
    if (!w) return fail(APS_ERR_ARG, "%s: NULL pointer", what);
    if (mis(w, 16)) return fail(APS_ERR_ARG, "%s: the weight must be 16-byte aligned", what);
    if (static_cast<int64_t>(to.out) * to.in > int64_t(1) << 38)
        return fail(APS_ERR_SHAPE, "%s: a weight of %d x %d", what, to.out, to.in);
    const size_t bytes = static_cast<size_t>(to.out) * to.in * (dtype == APS_DTYPE_F32 ? 4 : 2);
    const Q4Bytes b = q4_bytes(to);
    if (overlap_q4(w, bytes, to) || overlap(to.codes, b.codes, to.scales, b.scales) ||
        overlap(to.codes, b.codes, to.zeros, b.zeros) || overlap(to.scales, b.scales, to.zeros, b.zeros))
        return fail(APS_ERR_ARG, "%s: an output overlaps another array", what);
    return launched(aps::launch_quantise_q4(w, dtype == APS_DTYPE_F32, to.out, to.in, to.group,
                                            const_cast<uint8_t*>(to.codes), const_cast<void*>(to.scales),
                                            to.scales_f32, const_cast<uint8_t*>(to.zeros),
                                            static_cast<hipStream_t>(stream)),
                    "quantise_q4 launch");
}

size_t aps_token_logprobs_workspace_size(int64_t rows, int64_t vocab, int32_t top, int32_t dtype) {
    if (check_logprobs(rows, vocab, top, dtype, "token_logprobs")) return 0;
    return aps::token_logprobs_part_bytes(rows, vocab, top, dtype == APS_DTYPE_F32);
}

int aps_token_logprobs(const void* logits, int64_t logits_stride, int32_t dtype, int64_t rows, int64_t vocab,
                       const int32_t* tokens, int64_t n_tokens, int32_t top, float* logprobs, float* entropy,
                       int32_t* top_ids, float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "token_logprobs";
    if (int rc = check_logprobs(rows, vocab, top, dtype, what)) return rc;
    if (logits_stride < vocab)
        return fail(APS_ERR_SHAPE, "%s: row stride %lld of %lld logits", what, (long long)logits_stride,
                    (long long)vocab);
    if (n_tokens < 0 || n_tokens > kMaxRows || rows * n_tokens > int64_t(1) << 40)
        return fail(APS_ERR_SHAPE, "%s: %lld tokens a row", what, (long long)n_tokens);
    if (rows == 0) return APS_OK;
    if (!logits || (n_tokens && (!tokens || !logprobs)) || (top && (!top_ids || !top_logprobs)))
        return fail(APS_ERR_ARG, "%s: NULL pointer", what);
    if (mis(logits, dtype == APS_DTYPE_F32 ? 4 : 2) || mis(tokens, 4) || mis(logprobs, 4) || mis(entropy, 4) ||
        mis(top_ids, 4) || mis(top_logprobs, 4))
        return fail(APS_ERR_ARG, "%s: arrays must be aligned to their elements", what);
    const size_t need = aps::token_logprobs_part_bytes(rows, vocab, top, dtype == APS_DTYPE_F32);
    if (need && (!workspace || workspace_bytes < need))
        return fail(APS_ERR_WORKSPACE, "%s: workspace %zu bytes, need %zu", what, workspace_bytes, need);
    if (need && mis(workspace, 16)) return fail(APS_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", what);
    const int64_t n = rows * n_tokens * 4, t = rows * top * 4;
    // what is written, then what is read
    const Rows out[5] = {{logprobs, 1, n, n},
                         {entropy, entropy ? 1 : 0, 4 * rows, 4 * rows},
                         {top_ids, 1, t, t},
                         {top_logprobs, 1, t, t},
                         {workspace, 1, static_cast<int64_t>(need), static_cast<int64_t>(need)}};
    const Rows from = rows_of(logits, rows, vocab, logits_stride, dtype == APS_DTYPE_F32 ? 4 : 2);
    for (int i = 0; i < 5; ++i) {
        bool clash = overlap(out[i], from) || overlap(out[i], {tokens, 1, n, n});
        for (int j = 0; j < i; ++j) clash = clash || overlap(out[i], out[j]);
        if (clash) return fail(APS_ERR_ARG, "%s: an output overlaps another array", what);
    }
    const aps::LogprobArgs a{logits, logits_stride, rows,    vocab,        tokens, n_tokens, top, logprobs,
                             entropy, top_ids,      top_logprobs, static_cast<float*>(workspace)};
    return launched(aps::launch_token_logprobs(a, dtype == APS_DTYPE_F32, static_cast<hipStream_t>(stream)),
                    "token_logprobs launch");
}

}  // extern "C"
