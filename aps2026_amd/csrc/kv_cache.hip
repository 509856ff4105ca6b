// The paged key/value cache: aps_kv_append rotates the new tokens' queries and
// keys by their positions and writes keys and values into their pages;
// aps_kv_gather reads rows back.
//
// Rotation of the pair (x0, x1) = (x[j], x[j + D/2]) by the angle at the row's
// position: x0' = x0 c - x1 s, x1' = x0 s + x1 c.  In 64 bits the products of
// fp32 (or bf16) values with fp32 table entries are exact, so a result is
// rounded by the sum and then once to fp32: nothing depends on the order or on
// fused steps, and the 4-bit codes of a value next to a border are the same in
// every implementation of the formula.  The kernel is bound by its bytes, the
// four 64-bit operations of a pair hide behind them.
//
// D / 16 threads take one head of one row, 8 values of each half: 16-byte
// accesses (bf16), both halves of every pair in one thread, and the 32 values
// of a 4-bit block in four neighbouring lanes.
#include <algorithm>

#include "serve.hpp"

namespace aps {
namespace {

constexpr int kThreads = 256;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <bool F32, bool VEC>
__device__ inline void load8(const void* base, int64_t at, float (&x)[8]) {
    if constexpr (F32) {
        const float* p = static_cast<const float*>(base) + at;
        if constexpr (VEC) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p[i];
        }
    } else {
        const bf16_t* p = static_cast<const bf16_t*>(base) + at;
        if constexpr (VEC) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[2 * i] = bf16w_lo(w[i]); x[2 * i + 1] = bf16w_hi(w[i]); }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(static_cast<uint32_t>(p[i]) << 16);
        }
    }
}

template <bool F32, bool VEC>
__device__ inline void store8(void* base, int64_t at, const float (&x)[8]) {
    if constexpr (F32) {
        float* p = static_cast<float*>(base) + at;
        if constexpr (VEC) {
            *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = x[i];
        }
    } else {
        bf16_t* p = static_cast<bf16_t*>(base) + at;
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack2_bf16(x[2 * i], x[2 * i + 1]);
        if constexpr (VEC) {
            *reinterpret_cast<u32x4*>(p) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = static_cast<bf16_t>(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu);
        }
    }
}

// lo and hi: the 8 values of the lower and the upper half that this thread
// holds of one head (dims 8 t .. and D / 2 + 8 t ..), written at a slot.
template <int D, Kv KV>
__device__ inline void hold(void* base, uint8_t* scales, int64_t head_row, int t, const float (&lo)[8],
                            const float (&hi)[8]) {
    if constexpr (KV == Kv::kMx) {
        uint32_t am[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            am[0] = max(am[0], __float_as_uint(lo[i]) & 0x7FFFFFFFu);
            am[1] = max(am[1], __float_as_uint(hi[i]) & 0x7FFFFFFFu);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            am[h] = max(am[h], static_cast<uint32_t>(__shfl_xor(static_cast<int>(am[h]), 1)));
            am[h] = max(am[h], static_cast<uint32_t>(__shfl_xor(static_cast<int>(am[h]), 2)));
        }
        const uint32_t b0 = mx_scale_byte(am[0]), b1 = mx_scale_byte(am[1]);
        auto* codes = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(base) + head_row * (D / 2));
        codes[t] = mx_encode8(lo, mx_scale(b0));
        codes[D / 16 + t] = mx_encode8(hi, mx_scale(b1));
        if ((t & 3) == 0) {
            uint8_t* sc = scales + head_row * (D / 32);
            sc[t / 4] = static_cast<uint8_t>(b0);
            sc[D / 64 + t / 4] = static_cast<uint8_t>(b1);
        }
    } else {
        store8<KV == Kv::kF32, true>(base, head_row * D + 8 * t, lo);
        store8<KV == Kv::kF32, true>(base, head_row * D + D / 2 + 8 * t, hi);
    }
}

template <int D, bool SRC32, Kv KV, bool VEC>
__global__ void __launch_bounds__(kThreads)
k_kv_append(KvCache c, KvAppendArgs a) {
    constexpr int TPH = D / 16;  // threads of one head
    const uint32_t heads = static_cast<uint32_t>(2 * c.kv_heads + a.q_heads);
    const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / TPH;
    const int t = threadIdx.x % TPH;
    const int64_t row = item / heads;
    if (row >= a.rows) return;  // a head's threads leave together
    const int head = static_cast<int>(item - row * heads);
    const bool is_v = head >= c.kv_heads && head < 2 * c.kv_heads, is_q = head >= 2 * c.kv_heads;
    const int h = is_q ? head - 2 * c.kv_heads : is_v ? head - c.kv_heads : head;
    const int64_t slot = is_q ? 0 : a.slots[row];
    if (slot < 0 || slot >= c.num_pages << c.page_shift) return;
    const void* src = is_q ? a.q : is_v ? a.v : a.k;
    const int64_t at = row * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + static_cast<int64_t>(h) * D + 8 * t;
    float x0[8], x1[8];
    load8<SRC32, VEC>(src, at, x0);
    load8<SRC32, VEC>(src, at + D / 2, x1);
    const int64_t pos = a.positions[row];
    if (!is_v && pos >= 0 && pos < a.max_pos) {
        float co[8], si[8];
        load8<true, VEC>(a.cosv, pos * (D / 2) + 8 * t, co);
        load8<true, VEC>(a.sinv, pos * (D / 2) + 8 * t, si);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double u = x0[i], w = x1[i], cc = co[i], ss = si[i];
            x0[i] = static_cast<float>(u * cc - w * ss);
            x1[i] = static_cast<float>(u * ss + w * cc);
        }
    }
    if (is_q) {
        const int64_t to = row * a.q_out_stride + static_cast<int64_t>(h) * D + 8 * t;
        store8<SRC32, VEC>(a.q_out, to, x0);
        store8<SRC32, VEC>(a.q_out, to + D / 2, x1);
        return;
    }
    const int64_t page = slot >> c.page_shift, off = slot & ((1 << c.page_shift) - 1);
    const int64_t head_row = ((page * c.kv_heads + h) << c.page_shift) + off;
    hold<D, KV>(is_v ? c.v : c.k, is_v ? c.v_scale : c.k_scale, head_row, t, x0, x1);
}

template <int D, Kv KV, bool OUT32>
__global__ void __launch_bounds__(kThreads)
k_kv_gather(KvCache c, const int64_t* __restrict__ slots, int64_t rows, void* k_out, void* v_out) {
    constexpr int TPH = D / 8;
    const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / TPH;
    const int t = threadIdx.x % TPH;
    const int64_t row = item / c.kv_heads;
    if (row >= rows) return;
    const int h = static_cast<int>(item - row * c.kv_heads);
    const int64_t slot = slots[row];
    const bool live = slot >= 0 && slot < c.num_pages << c.page_shift;
    const int64_t page = slot >> c.page_shift, off = slot & ((1 << c.page_shift) - 1);
    const int64_t head_row = live ? ((page * c.kv_heads + h) << c.page_shift) + off : 0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        void* out = which ? v_out : k_out;
        if (!out) continue;
        const void* base = which ? c.v : c.k;
        float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (live) {
            if constexpr (KV == Kv::kMx) {
                const uint32_t w = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) +
                                                                     head_row * (D / 2))[t];
                const float sc = mx_scale((which ? c.v_scale : c.k_scale)[head_row * (D / 32) + t / 4]);
                const uint32_t p[4] = {mx_decode2<0>(w, sc), mx_decode2<1>(w, sc), mx_decode2<2>(w, sc),
                                       mx_decode2<3>(w, sc)};
#pragma unroll
                for (int i = 0; i < 4; ++i) { x[2 * i] = bf16w_lo(p[i]); x[2 * i + 1] = bf16w_hi(p[i]); }
            } else {
                load8<KV == Kv::kF32, true>(base, head_row * D + 8 * t, x);
            }
        }
        store8<OUT32, true>(out, (row * c.kv_heads + h) * D + 8 * t, x);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int D, bool SRC32, Kv KV>
void append(const KvCache& c, const KvAppendArgs& a, unsigned blocks, bool vec, hipStream_t s) {
    if (vec) hipLaunchKernelGGL((k_kv_append<D, SRC32, KV, true>), dim3(blocks), dim3(kThreads), 0, s, c, a);
    else hipLaunchKernelGGL((k_kv_append<D, SRC32, KV, false>), dim3(blocks), dim3(kThreads), 0, s, c, a);
}

template <int D>
hipError_t append_d(const KvCache& c, const KvAppendArgs& all, bool src_f32, hipStream_t s) {
    const int64_t per = src_f32 ? 4 : 8;  // elements of 16 bytes
    const bool vec = aligned16(all.k) && aligned16(all.v) && aligned16(all.q) && aligned16(all.q_out) &&
                     aligned16(all.cosv) && aligned16(all.sinv) && all.k_stride % per == 0 && all.v_stride % per == 0 &&
                     (all.q_heads == 0 || (all.q_stride % per == 0 && all.q_out_stride % per == 0));
    const int64_t threads = static_cast<int64_t>(2 * c.kv_heads + all.q_heads) * (D / 16);   // of a row
    const int64_t most = most_blocks(kThreads) * kThreads / threads, size = src_f32 ? 4 : 2;
    for (int64_t first = 0; first < all.rows; first += most) {
        KvAppendArgs a = all;
        a.rows = std::min(most, all.rows - first);
        a.positions += first;
        a.slots += first;
        a.k = static_cast<const char*>(all.k) + first * all.k_stride * size;
        a.v = static_cast<const char*>(all.v) + first * all.v_stride * size;
        if (all.q_heads > 0) {
            a.q = static_cast<const char*>(all.q) + first * all.q_stride * size;
            a.q_out = static_cast<char*>(all.q_out) + first * all.q_out_stride * size;
        }
        const unsigned n = static_cast<unsigned>(ceil_div(a.rows * threads, kThreads));
        if (c.type == Kv::kF32) append<D, true, Kv::kF32>(c, a, n, vec, s);
        else if (c.type == Kv::kBf16 && src_f32) append<D, true, Kv::kBf16>(c, a, n, vec, s);
        else if (c.type == Kv::kBf16) append<D, false, Kv::kBf16>(c, a, n, vec, s);
        else if (src_f32) append<D, true, Kv::kMx>(c, a, n, vec, s);
        else append<D, false, Kv::kMx>(c, a, n, vec, s);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int D, Kv KV>
void gather(const KvCache& c, const int64_t* slots, int64_t rows, void* k, void* v, bool f32, unsigned n,
            hipStream_t s) {
    if (f32) hipLaunchKernelGGL((k_kv_gather<D, KV, true>), dim3(n), dim3(kThreads), 0, s, c, slots, rows, k, v);
    else hipLaunchKernelGGL((k_kv_gather<D, KV, false>), dim3(n), dim3(kThreads), 0, s, c, slots, rows, k, v);
}

template <int D>
hipError_t gather_d(const KvCache& c, const int64_t* slots, int64_t all, void* k_out, void* v_out, bool f32, hipStream_t s) {
    const int64_t threads = static_cast<int64_t>(c.kv_heads) * (D / 8);   // of a row
    const int64_t most = most_blocks(kThreads) * kThreads / threads, bytes = static_cast<int64_t>(c.kv_heads) * D * (f32 ? 4 : 2);
    for (int64_t first = 0; first < all; first += most) {
        const int64_t rows = std::min(most, all - first), *at = slots + first;
        void* k = k_out ? static_cast<char*>(k_out) + first * bytes : nullptr;
        void* v = v_out ? static_cast<char*>(v_out) + first * bytes : nullptr;
        const unsigned n = static_cast<unsigned>(ceil_div(rows * threads, kThreads));
        if (c.type == Kv::kF32) gather<D, Kv::kF32>(c, at, rows, k, v, f32, n, s);
        else if (c.type == Kv::kBf16) gather<D, Kv::kBf16>(c, at, rows, k, v, f32, n, s);
        else gather<D, Kv::kMx>(c, at, rows, k, v, f32, n, s);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_kv_append(const KvCache& cache, const KvAppendArgs& a, bool src_f32, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    return cache.head_dim == 128 ? append_d<128>(cache, a, src_f32, s) : append_d<64>(cache, a, src_f32, s);
}

hipError_t launch_kv_gather(const KvCache& cache, const int64_t* slots, int64_t rows, void* k_out, void* v_out,
                            bool out_f32, hipStream_t s) {
    if (rows <= 0 || (!k_out && !v_out)) return hipSuccess;
    return cache.head_dim == 128 ? gather_d<128>(cache, slots, rows, k_out, v_out, out_f32, s)
                                 : gather_d<64>(cache, slots, rows, k_out, v_out, out_f32, s);
}

}  // namespace aps
