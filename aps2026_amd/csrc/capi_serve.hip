// C ABI of the serving operators (declared in include/aps_serve.h): argument
// checks, then the launches.
#include "../../include/aps_serve.h"
#include "serve.hpp"

namespace {

using aps::fail;

constexpr int64_t kMaxRows = int64_t(1) << 30;
constexpr int64_t kMaxBatch = int64_t(1) << 20;  // workgroups look their sequence up among all of them

bool mis(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

bool overlap(const void* p, size_t np, const void* q, size_t nq) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return np && nq && a < b + nq && b < a + np;
}

// `count` rows of `width` bytes, `stride` bytes apart.
typedef __int128 wide;
struct Rows {
    const void* at;
    int64_t count, width;
    wide stride;
};
Rows rows_of(const void* p, int64_t rows, int64_t values, int64_t stride, uintptr_t elt) {
    const int64_t e = static_cast<int64_t>(elt);
    return {p, p ? rows : 0, values * e, static_cast<wide>(stride) * e};
}
// True if a row of a shares a byte with a row of b: of slices of one wider row,
// which lie between each other, none does.
bool overlap(const Rows& a, const Rows& b) {
    if (a.count <= 0 || b.count <= 0 || a.width <= 0 || b.width <= 0) return false;
    const wide d = static_cast<wide>(reinterpret_cast<uintptr_t>(b.at)) - reinterpret_cast<uintptr_t>(a.at);
    if (d >= (a.count - 1) * a.stride + a.width ||
        -d >= (b.count - 1) * b.stride + b.width)
        return false;
    if (a.count == 1 && b.count == 1) return true;
    auto floor_div = [](wide x, wide y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
    // the first row of b that ends behind the start of a's row i, from
    // b.width + d + j stride > i stride; rows of one stride are alike for all i
    if (a.stride == b.stride || a.count == 1 || b.count == 1) {
        // (a single row's stride is the other's)
        const wide s = a.count == 1 ? b.stride : a.stride;
        const wide first = -(a.count - 1), last = b.count - 1;
        wide j = floor_div(-d - b.width, s) + 1;
        if (j < first) j = first;
        return j <= last && d + j * s < a.width;
    }
    for (int64_t i = 0; i < a.count; ++i) {
        const wide to = i * a.stride;
        wide j = floor_div(to - d - b.width, b.stride) + 1;
        if (j < 0) j = 0;
        if (j < b.count && d + j * b.stride < to + a.width) return true;
    }
    return false;
}

int launched(hipError_t err, const char* what) {
    if (err == hipSuccess) return APS_OK;
    return fail(APS_ERR_HIP, "%s: %s", what, hipGetErrorString(err));
}

// The cache description; with `arrays` its pointers too.
int check_cache(const aps_kv_cache* d, const char* what, bool arrays, aps::KvCache* out) {
    if (!d) return fail(APS_ERR_ARG, "%s: NULL cache", what);
    if (d->dtype != APS_DTYPE_F32 && d->dtype != APS_DTYPE_BF16 && d->dtype != APS_KV_MXFP4)
        return fail(APS_ERR_DTYPE, "%s: cache dtype %d", what, d->dtype);
    int shift = 0;
    while (shift < 8 && (1 << shift) < d->page_size) ++shift;
    if (shift < 4 || (1 << shift) != d->page_size)
        return fail(APS_ERR_SHAPE, "%s: page size %d (16, 32, 64, 128 or 256)", what, d->page_size);
    if (d->head_dim != 64 && d->head_dim != 128)
        return fail(APS_ERR_SHAPE, "%s: head_dim %d (64 or 128)", what, d->head_dim);
    if (d->kv_heads < 1 || d->kv_heads > 4096) return fail(APS_ERR_SHAPE, "%s: %d key heads", what, d->kv_heads);
    if (d->num_pages < 1 || d->num_pages > (int64_t(1) << 40) / d->page_size)
        return fail(APS_ERR_SHAPE, "%s: %lld pages", what, (long long)d->num_pages);
    const bool mx = d->dtype == APS_KV_MXFP4;
    if (arrays) {
        if (!d->k || !d->v || (mx && (!d->k_scale || !d->v_scale)))
            return fail(APS_ERR_ARG, "%s: NULL cache array", what);
        if (mis(d->k, 16) || mis(d->v, 16) || (mx && (mis(d->k_scale, 4) || mis(d->v_scale, 4))))
            return fail(APS_ERR_ARG, "%s: cache arrays must be 16-byte (scales 4-byte) aligned", what);
    }
    out->k = d->k;
    out->v = d->v;
    out->k_scale = mx ? static_cast<uint8_t*>(d->k_scale) : nullptr;
    out->v_scale = mx ? static_cast<uint8_t*>(d->v_scale) : nullptr;
    out->num_pages = d->num_pages;
    out->page_shift = shift;
    out->kv_heads = d->kv_heads;
    out->head_dim = d->head_dim;
    out->type = static_cast<aps::Kv>(d->dtype);
    return APS_OK;
}

// Bytes of k, and of v.
int64_t held_bytes(const aps::KvCache& c) {
    const int64_t n = (c.num_pages << c.page_shift) * c.kv_heads * c.head_dim;
    return c.type == aps::Kv::kMx ? n / 2 : c.type == aps::Kv::kBf16 ? 2 * n : 4 * n;
}

int check_heads(const aps::KvCache& c, int32_t q_heads, const char* what) {
    if (q_heads < 1 || q_heads > 65536 || q_heads % c.kv_heads != 0)
        return fail(APS_ERR_SHAPE, "%s: %d query heads on %d key heads", what, q_heads, c.kv_heads);
    return APS_OK;
}

int check_source(const aps::KvCache& c, int32_t dtype, const char* what) {
    if (dtype != APS_DTYPE_F32 && dtype != APS_DTYPE_BF16) return fail(APS_ERR_DTYPE, "%s: dtype %d", what, dtype);
    if (c.type == aps::Kv::kF32 && dtype != APS_DTYPE_F32)
        return fail(APS_ERR_DTYPE, "%s: an fp32 cache takes fp32 tensors", what);
    return APS_OK;
}

int check_paged(const aps::KvCache& c, int64_t rows, int32_t q_heads, int64_t batch, int64_t max_q_len,
                int64_t max_kv_len, int32_t window, int32_t sinks, aps::PagedArgs* a) {
    const char* what = "attention_paged";
    if (int rc = check_heads(c, q_heads, what)) return rc;
    if (rows < 0 || rows > kMaxRows || batch < 0 || batch > kMaxBatch || max_q_len < 0 || max_kv_len < 0 ||
        max_kv_len > kMaxRows)
        return fail(APS_ERR_SHAPE, "%s: rows %lld, batch %lld, max_q_len %lld, max_kv_len %lld", what, (long long)rows,
                    (long long)batch, (long long)max_q_len, (long long)max_kv_len);
    if (rows * q_heads > int64_t(1) << 40)  // sizes in bytes stay far from 64 bits
        return fail(APS_ERR_SHAPE, "%s: %lld rows of %d heads", what, (long long)rows, q_heads);
    if (window < 1 || sinks < 0) return fail(APS_ERR_SHAPE, "%s: window %d, sinks %d", what, window, sinks);
    a->rows = rows;
    a->q_heads = q_heads;
    a->batch = batch;
    // a sequence has no more queries than there are rows
    a->max_q_len = max_q_len < rows ? max_q_len : rows;
    a->max_kv_len = max_kv_len;
    a->window = window;
    a->sinks = sinks;
    if (a->max_q_len * (q_heads / c.kv_heads) > kMaxRows)
        return fail(APS_ERR_SHAPE, "%s: %lld rows under a key head", what,
                    (long long)(a->max_q_len * (q_heads / c.kv_heads)));
    if (rows == 0 || batch == 0 || a->max_q_len == 0) return APS_OK;
    const int64_t blocks = aps::attention_paged_blocks(c, *a);
    if (blocks > 0x7FFFFFFF) return fail(APS_ERR_SHAPE, "%s: %lld workgroups", what, (long long)blocks);
    return APS_OK;
}

}  // namespace

extern "C" {

int aps_kv_append(const aps_kv_cache* cache, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                  const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, int32_t src_dtype, int64_t rows,
                  int32_t q_heads, const int32_t* positions, const int64_t* slots, const float* cos_table,
                  const float* sin_table, int64_t max_pos, void* stream) {
    const char* what = "kv_append";
    aps::KvCache c;
    if (int rc = check_cache(cache, what, rows > 0, &c)) return rc;
    if (int rc = check_source(c, src_dtype, what)) return rc;
    if (rows < 0 || rows > kMaxRows || max_pos < 0 || max_pos > kMaxRows)
        return fail(APS_ERR_SHAPE, "%s: rows %lld, max_pos %lld", what, (long long)rows, (long long)max_pos);
    const int64_t kv = static_cast<int64_t>(c.kv_heads) * c.head_dim;
    if (k_stride < kv || v_stride < kv)
        return fail(APS_ERR_SHAPE, "%s: row strides %lld, %lld of %lld values", what, (long long)k_stride,
                    (long long)v_stride, (long long)kv);
    if (q) {
        if (int rc = check_heads(c, q_heads, what)) return rc;
        const int64_t qd = static_cast<int64_t>(q_heads) * c.head_dim;
        if (q_stride < qd || q_out_stride < qd)
            return fail(APS_ERR_SHAPE, "%s: query row strides %lld, %lld of %lld values", what, (long long)q_stride,
                        (long long)q_out_stride, (long long)qd);
        if (q == q_out && q_stride != q_out_stride)
            return fail(APS_ERR_ARG, "%s: queries rotated in place keep their stride", what);
    }
    if (rows == 0) return APS_OK;
    const uintptr_t elt = src_dtype == APS_DTYPE_F32 ? 4 : 2;
    if (!k || !v || !positions || !slots || (max_pos > 0 && (!cos_table || !sin_table)) || (q && !q_out))
        return fail(APS_ERR_ARG, "%s: NULL pointer", what);
    // a row is read after others were written
    const int64_t qd = static_cast<int64_t>(q_heads) * c.head_dim;
    const Rows to = rows_of(q ? q_out : nullptr, rows, qd, q_out_stride, elt);
    const int64_t held = held_bytes(c);
    if ((q != q_out && overlap(to, rows_of(q, rows, qd, q_stride, elt))) ||
        overlap(to, rows_of(k, rows, kv, k_stride, elt)) || overlap(to, rows_of(v, rows, kv, v_stride, elt)) ||
        overlap(to, {c.k, 1, held, held}) || overlap(to, {c.v, 1, held, held}))
        return fail(APS_ERR_ARG, "%s: q_out overlaps another array", what);
    if (mis(k, elt) || mis(v, elt) || mis(q, elt) || mis(q_out, elt) || mis(positions, 4) || mis(slots, 8) ||
        mis(cos_table, 4) || mis(sin_table, 4))
        return fail(APS_ERR_ARG, "%s: arrays must be aligned to their elements", what);
    aps::KvAppendArgs a{k,         v,        q,    q ? q_out : nullptr, k_stride, v_stride,  q_stride,  q_out_stride,
                        rows,      q ? q_heads : 0, positions, slots,   cos_table, sin_table, max_pos};
    return launched(aps::launch_kv_append(c, a, src_dtype == APS_DTYPE_F32, static_cast<hipStream_t>(stream)),
                    "kv_append launch");
}

int aps_kv_gather(const aps_kv_cache* cache, const int64_t* slots, int64_t rows, void* k_out, void* v_out,
                  int32_t out_dtype, void* stream) {
    const char* what = "kv_gather";
    aps::KvCache c;
    if (int rc = check_cache(cache, what, rows > 0, &c)) return rc;
    if (out_dtype != APS_DTYPE_F32 && out_dtype != APS_DTYPE_BF16)
        return fail(APS_ERR_DTYPE, "%s: dtype %d", what, out_dtype);
    if (rows < 0 || rows > kMaxRows) return fail(APS_ERR_SHAPE, "%s: rows %lld", what, (long long)rows);
    if (rows == 0 || (!k_out && !v_out)) return APS_OK;
    if (!slots) return fail(APS_ERR_ARG, "%s: NULL pointer", what);
    const int64_t kv = static_cast<int64_t>(c.kv_heads) * c.head_dim, held = held_bytes(c);
    const size_t out_bytes = static_cast<size_t>(rows * kv) * (out_dtype == APS_DTYPE_F32 ? 4 : 2);
    for (void* to : {k_out, v_out})
        if (to && (overlap(to, out_bytes, c.k, held) || overlap(to, out_bytes, c.v, held) ||
                   overlap(to, out_bytes, to == k_out ? v_out : nullptr, v_out ? out_bytes : 0)))
            return fail(APS_ERR_ARG, "%s: an output overlaps another array", what);
    if (mis(k_out, 16) || mis(v_out, 16) || mis(slots, 8))
        return fail(APS_ERR_ARG, "%s: outputs must be 16-byte, slots 8-byte aligned", what);
    return launched(aps::launch_kv_gather(c, slots, rows, k_out, v_out, out_dtype == APS_DTYPE_F32,
                                          static_cast<hipStream_t>(stream)),
                    "kv_gather launch");
}

size_t aps_attention_paged_workspace_size(const aps_kv_cache* cache, int64_t rows, int32_t q_heads, int64_t batch,
                                          int64_t max_q_len, int64_t max_kv_len, int32_t window, int32_t sinks) {
    aps::KvCache c;
    aps::PagedArgs a{};
    if (check_cache(cache, "attention_paged", false, &c)) return 0;
    if (check_paged(c, rows, q_heads, batch, max_q_len, max_kv_len, window, sinks, &a)) return 0;
    if (rows == 0 || batch == 0 || a.max_q_len == 0) return 0;
    return aps::attention_paged_part_bytes(c, a);
}

int aps_attention_paged(const aps_kv_cache* cache, const void* q, int64_t q_stride, int32_t q_dtype, int64_t rows,
                        int32_t q_heads, const int32_t* q_offsets, const int32_t* kv_lens, const int32_t* page_table,
                        int64_t table_stride, int64_t batch, int64_t max_q_len, int64_t max_kv_len, int32_t window,
                        int32_t sinks, float scale, void* out, void* workspace, size_t workspace_bytes,
                        void* stream) {
    const char* what = "attention_paged";
    aps::KvCache c;
    aps::PagedArgs a{};
    if (int rc = check_cache(cache, what, rows > 0 && batch > 0, &c)) return rc;
    if (int rc = check_source(c, q_dtype, what)) return rc;
    if (int rc = check_paged(c, rows, q_heads, batch, max_q_len, max_kv_len, window, sinks, &a)) return rc;
    const float scale_log2 = scale * aps::kLog2e;  // what the kernels take
    if (!(scale_log2 - scale_log2 == 0.0f)) return fail(APS_ERR_ARG, "%s: scale is not finite", what);
    const int64_t qd = static_cast<int64_t>(q_heads) * c.head_dim, per = q_dtype == APS_DTYPE_F32 ? 4 : 8;
    if (q_stride < qd || q_stride % per != 0)
        return fail(APS_ERR_SHAPE, "%s: query row stride %lld of %lld values", what, (long long)q_stride,
                    (long long)qd);
    if (table_stride < 0 || table_stride > kMaxRows)
        return fail(APS_ERR_SHAPE, "%s: table stride %lld", what, (long long)table_stride);
    if (rows == 0 || batch == 0 || a.max_q_len == 0) return APS_OK;
    if (!q || !out || !q_offsets || !kv_lens || (table_stride > 0 && !page_table))
        return fail(APS_ERR_ARG, "%s: NULL pointer", what);
    if (mis(q, 16) || mis(out, 16)) return fail(APS_ERR_ARG, "%s: q and out must be 16-byte aligned", what);
    if (mis(q_offsets, 4) || mis(kv_lens, 4) || mis(page_table, 4))
        return fail(APS_ERR_ARG, "%s: index arrays must be 4-byte aligned", what);
    const size_t need = aps::attention_paged_part_bytes(c, a);
    if (need && (!workspace || workspace_bytes < need))
        return fail(APS_ERR_WORKSPACE, "%s: workspace %zu bytes, need %zu", what, workspace_bytes, need);
    if (need && mis(workspace, 256)) return fail(APS_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", what);
    // rows are read after others were written: nothing in place
    const size_t elt = q_dtype == APS_DTYPE_F32 ? 4 : 2, out_bytes = static_cast<size_t>(rows * qd) * elt;
    const size_t q_bytes = static_cast<size_t>((rows - 1) * q_stride + qd) * elt;
    if (overlap(out, out_bytes, q, q_bytes) || overlap(workspace, need, out, out_bytes) ||
        overlap(workspace, need, q, q_bytes))
        return fail(APS_ERR_ARG, "%s: q, out and workspace overlap", what);
    a.q = q;
    a.q_stride = q_stride;
    a.q_offsets = q_offsets;
    a.kv_lens = kv_lens;
    a.page_table = page_table;
    a.table_stride = table_stride;
    a.scale = scale;
    a.out = out;
    a.part = static_cast<float*>(workspace);
    return launched(aps::launch_attention_paged(c, a, q_dtype == APS_DTYPE_F32, static_cast<hipStream_t>(stream)),
                    "attention_paged launch");
}

int aps_logits_process(const void* logits, int64_t logits_stride, int32_t dtype, int64_t rows, int64_t vocab,
                       const aps_logits_rules* rules, void* out, int64_t out_stride, void* stream) {
    const char* what = "logits_process";
    if (dtype != APS_DTYPE_F32 && dtype != APS_DTYPE_BF16) return fail(APS_ERR_DTYPE, "%s: dtype %d", what, dtype);
    if (!rules) return fail(APS_ERR_ARG, "%s: NULL rules", what);
    if (rows < 0 || rows > kMaxRows || vocab < 0 || vocab > kMaxRows)
        return fail(APS_ERR_SHAPE, "%s: rows %lld, vocab %lld", what, (long long)rows, (long long)vocab);
    if (logits_stride < vocab || out_stride < vocab)
        return fail(APS_ERR_SHAPE, "%s: row strides %lld, %lld of %lld logits", what, (long long)logits_stride,
                    (long long)out_stride, (long long)vocab);
    const aps_logits_rules& r = *rules;
    if (r.history && (!r.history_lens || r.history_stride < 0))
        return fail(APS_ERR_ARG, "%s: a history needs its lengths and its stride", what);
    if (r.bias_ids && (!r.bias_values || !r.bias_lens || r.bias_stride < 0))
        return fail(APS_ERR_ARG, "%s: biases need their values, lengths and stride", what);
    if (r.mask && (r.mask_rows < 0 || r.mask_stride < (vocab + 31) / 32))
        return fail(APS_ERR_SHAPE, "%s: mask rows of %lld words for %lld logits", what, (long long)r.mask_stride,
                    (long long)vocab);
    if (r.mask && !r.mask_index && r.mask_rows < rows)
        return fail(APS_ERR_SHAPE, "%s: %lld masks for %lld rows", what, (long long)r.mask_rows, (long long)rows);
    if (rows == 0 || vocab == 0) return APS_OK;
    if (!logits || !out) return fail(APS_ERR_ARG, "%s: NULL pointer", what);
    if (logits == out && logits_stride != out_stride)
        return fail(APS_ERR_ARG, "%s: logits changed in place keep their stride", what);
    const uintptr_t elt = dtype == APS_DTYPE_F32 ? 4 : 2;
    if (logits != out && overlap(rows_of(logits, rows, vocab, logits_stride, elt),
                                 rows_of(out, rows, vocab, out_stride, elt)))
        return fail(APS_ERR_ARG, "%s: logits and out overlap", what);
    if (mis(logits, elt) || mis(out, elt) || mis(r.history, 4) || mis(r.history_lens, 4) || mis(r.prompt_lens, 4) ||
        mis(r.repetition, 4) || mis(r.frequency, 4) || mis(r.presence, 4) || mis(r.bias_ids, 4) ||
        mis(r.bias_values, 4) || mis(r.bias_lens, 4) || mis(r.mask, 4) || mis(r.mask_index, 4))
        return fail(APS_ERR_ARG, "%s: arrays must be aligned to their elements", what);
    const aps::LogitsArgs a{logits,        out,           logits_stride, out_stride,    rows,         vocab,
                            r.history,     r.history_lens, r.prompt_lens, r.history_stride, r.repetition, r.frequency,
                            r.presence,    r.bias_ids,    r.bias_values, r.bias_lens,   r.bias_stride, r.mask,
                            r.mask_rows,   r.mask_stride, r.mask_index};
    return launched(aps::launch_logits_process(a, dtype == APS_DTYPE_F32, static_cast<hipStream_t>(stream)),
                    "logits_process launch");
}

}  // extern "C"
