// The rules on the logits of the next token (aps_logits_process): penalties
// for tokens already in the row's text, token biases and a grammar's mask.
//
// A workgroup takes a slice of one row's vocabulary.  It counts the history's
// tokens that fall into the slice in LDS (integer atomics, whose order changes
// nothing: the top bit marks a token seen in the prompt, the rest counts it
// past the prompt) and finds the bias of each token as the largest index of
// the list that names it, so that of an id named twice the last counts
// whatever the order.  Then it passes over the slice's logits once.  Bound by
// the logits' bytes; every slice reads the whole history, from L2 after the
// first.
#include <algorithm>

#include "serve.hpp"

namespace aps {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kSeenInPrompt = 0x80000000u;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <bool F32>
__device__ inline float load1(const void* p, int64_t i) {
    if constexpr (F32) return static_cast<const float*>(p)[i];
    else return __uint_as_float(static_cast<uint32_t>(static_cast<const bf16_t*>(p)[i]) << 16);
}
template <bool F32>
__device__ inline void store1(void* p, int64_t i, float v) {
    if constexpr (F32) static_cast<float*>(p)[i] = v;
    else static_cast<bf16_t*>(p)[i] = static_cast<bf16_t>(pack2_bf16(v, 0.0f) & 0xFFFFu);
}

// Four neighbouring logits.
template <bool F32>
__device__ inline void load4(const void* p, int64_t i, float (&x)[4]) {
    if constexpr (F32) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = v[k];
    } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const bf16_t*>(p) + i);
        x[0] = bf16w_lo(w[0]); x[1] = bf16w_hi(w[0]); x[2] = bf16w_lo(w[1]); x[3] = bf16w_hi(w[1]);
    }
}
template <bool F32>
__device__ inline void store4(void* p, int64_t i, const float (&x)[4]) {
    if constexpr (F32)
        *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = f32x4{x[0], x[1], x[2], x[3]};
    else
        *reinterpret_cast<u32x2*>(static_cast<bf16_t*>(p) + i) = u32x2{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
}

// VEC: rows of x and out start at 16 (bf16: 8) bytes' alignment, four logits
// to an access; they are read before the history, whose pass hides their way.
template <bool F32, bool VEC, int SLICE>
__global__ void __launch_bounds__(kThreads)
k_logits_process(LogitsArgs a, uint32_t slices, uint32_t deal) {
    constexpr int N = SLICE / (4 * kThreads);  // fours of a thread
    __shared__ __align__(16) uint32_t count[SLICE];
    __shared__ __align__(16) uint32_t bias[SLICE];
    const uint32_t turn = blockIdx.x / deal;
    const int64_t row = static_cast<int64_t>(turn / slices) * deal + blockIdx.x % deal;
    if (row >= a.rows) return;
    const int64_t base = static_cast<int64_t>(turn % slices) * SLICE;
    const int n = static_cast<int>(a.vocab - base < SLICE ? a.vocab - base : SLICE);
    const int tid = threadIdx.x;
    const bool hist = a.history != nullptr, biased = a.bias_ids != nullptr;
    const int64_t xr = row * a.x_stride + base, orow = row * a.out_stride + base;
    const uint32_t* mask = nullptr;
    if (a.mask) {
        const int64_t m = a.mask_index ? a.mask_index[row] : row;
        if (m >= 0 && m < a.mask_rows) mask = a.mask + m * a.mask_stride;
    }
    // the row's numbers before the logits: nothing waits for them later
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float freq = a.frequency ? a.frequency[row] : 0.0f;
    const float pres = a.presence ? a.presence[row] : 0.0f;
    const int64_t seen_len = hist ? min(static_cast<int64_t>(a.history_lens[row]), a.history_stride) : 0;
    const int64_t prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
    const int64_t bias_len = biased ? min(static_cast<int64_t>(a.bias_lens[row]), a.bias_stride) : 0;
    float x[N][4];
    uint32_t bits[N];
    if constexpr (VEC) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = 4 * (tid + kThreads * k);
            bits[k] = 15u;
            if (i + 4 <= n) {
                load4<F32>(a.x, xr + i, x[k]);
                if (mask) bits[k] = mask[(base + i) >> 5] >> (i & 31);
            }
        }
    }
    if (hist) {
        for (int i = 4 * tid; i < SLICE; i += 4 * kThreads) *reinterpret_cast<u32x4*>(count + i) = u32x4{0u, 0u, 0u, 0u};
    }
    if (biased) {
        for (int i = 4 * tid; i < SLICE; i += 4 * kThreads) *reinterpret_cast<u32x4*>(bias + i) = u32x4{0u, 0u, 0u, 0u};
    }
    if (hist || biased) __syncthreads();
    if (hist) {
        const int64_t len = seen_len;
        const int32_t* ids = a.history + row * a.history_stride;
        auto see = [&](int64_t i, int32_t id) {
            const uint32_t t = static_cast<uint32_t>(id) - static_cast<uint32_t>(base);  // a negative id is past 2^31
            if (t >= static_cast<uint32_t>(n)) return;
            if (i < prompt) atomicOr(&count[t], kSeenInPrompt);
            else atomicAdd(&count[t], 1u);
        };
        int64_t i = tid;
        for (; i + 3 * kThreads < len; i += 4 * kThreads) {
            int32_t id[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) id[k] = ids[i + k * kThreads];
#pragma unroll
            for (int k = 0; k < 4; ++k) see(i + k * kThreads, id[k]);
        }
        for (; i < len; i += kThreads) see(i, ids[i]);
    }
    if (biased) {
        const int64_t len = bias_len;
        const int32_t* ids = a.bias_ids + row * a.bias_stride;
        for (int64_t i = tid; i < len; i += kThreads) {
            const uint32_t t = static_cast<uint32_t>(ids[i]) - static_cast<uint32_t>(base);
            if (t < static_cast<uint32_t>(n)) atomicMax(&bias[t], static_cast<uint32_t>(i + 1));
        }
    }
    if (hist || biased) __syncthreads();
    const float* bv = a.bias_values + row * a.bias_stride;
    auto rule = [&](float v, uint32_t cnt, uint32_t bi, bool allowed) {
        if (cnt) v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
        const uint32_t times = cnt & ~kSeenInPrompt;
        if (times) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, static_cast<float>(times))), pres);
        if (bi) v = __fadd_rn(v, bv[bi - 1]);
        return allowed ? v : -INFINITY;
    };
    auto one = [&](int k) {
        store1<F32>(a.out, orow + k, rule(load1<F32>(a.x, xr + k), hist ? count[k] : 0u, biased ? bias[k] : 0u,
                                          !mask || ((mask[(base + k) >> 5] >> (k & 31)) & 1u)));
    };
    if constexpr (VEC) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = 4 * (tid + kThreads * k);
            if (i + 4 <= n) {
                u32x4 cnt{0u, 0u, 0u, 0u}, bi{0u, 0u, 0u, 0u};
                if (hist) cnt = *reinterpret_cast<const u32x4*>(count + i);
                if (biased) bi = *reinterpret_cast<const u32x4*>(bias + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[k][j] = rule(x[k][j], cnt[j], bi[j], (bits[k] >> j) & 1u);
                store4<F32>(a.out, orow + i, x[k]);
            } else {
                for (int j = i; j < n; ++j) one(j);
            }
        }
    } else {
        for (int k = tid; k < n; k += kThreads) one(k);
    }
}

// `rows` of the rows from `first` on.
LogitsArgs rows_from(LogitsArgs a, int64_t first, int64_t rows, int64_t size) {
    auto skip = [&](auto& p, int64_t values) { if (p) p += first * values; };
    a.rows = rows;
    a.x = static_cast<const char*>(a.x) + first * a.x_stride * size;
    a.out = static_cast<char*>(a.out) + first * a.out_stride * size;
    skip(a.history, a.history_stride);
    skip(a.history_lens, 1);
    skip(a.prompt_lens, 1);
    skip(a.repetition, 1);
    skip(a.frequency, 1);
    skip(a.presence, 1);
    skip(a.bias_ids, a.bias_stride);
    skip(a.bias_values, a.bias_stride);
    skip(a.bias_lens, 1);
    if (a.mask_index) {
        a.mask_index += first;
    } else if (a.mask) {
        a.mask += first * a.mask_stride;
        a.mask_rows -= first;
    }
    return a;
}

template <bool F32, int SLICE>
hipError_t launch(const LogitsArgs& a, bool vec, hipStream_t s) {
    // workgroups go round the XCDs: rows dealt the same way keep the slices of one
    // on an XCD, whose L2 then fetches its history once (256 x 32064, history 2048:
    // 47.8 -> 35.7 MB, 20.7 -> 18.6 us).  Of 8 to 128 rows either order takes the
    // same to within 0.2 us, and fewer than 8 would leave XCDs idle.
    const int64_t deal = a.rows >= 64 ? 8 : 1;
    const int64_t slices = ceil_div(a.vocab, SLICE), most = most_blocks(kThreads) / slices / deal * deal;
    const uint32_t n = static_cast<uint32_t>(slices), m = static_cast<uint32_t>(deal);
    for (int64_t first = 0; first < a.rows; first += most) {
        const LogitsArgs part = rows_from(a, first, std::min(most, a.rows - first), F32 ? 4 : 2);
        const dim3 grid(static_cast<unsigned>(ceil_div(part.rows, deal) * deal * slices)), block(kThreads);
        if (vec) hipLaunchKernelGGL((k_logits_process<F32, true, SLICE>), grid, block, 0, s, part, n, m);
        else hipLaunchKernelGGL((k_logits_process<F32, false, SLICE>), grid, block, 0, s, part, n, m);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_logits_process(const LogitsArgs& a, bool f32, hipStream_t s) {
    if (a.rows <= 0 || a.vocab <= 0) return hipSuccess;
    const uintptr_t mis = (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out)) & (f32 ? 15u : 7u);
    const bool vec = mis == 0 && a.x_stride % 4 == 0 && a.out_stride % 4 == 0;
    // Slices of 1024 until slices of 2048 give every CU one: a short launch ends
    // sooner (1 x 32064, history 613: 4.3 us, 4096 wide 5.5); wider ones read the
    // history less often (256 x 32064, history 2048: 1024 wide 23.2 us,
    // 2048 18.7, 4096 21.8).
    if (a.rows * ceil_div(a.vocab, 2048) < 256)
        return f32 ? launch<true, 1024>(a, vec, s) : launch<false, 1024>(a, vec, s);
    return f32 ? launch<true, 2048>(a, vec, s) : launch<false, 2048>(a, vec, s);
}

}  // namespace aps
