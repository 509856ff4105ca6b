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

// VEC: rows of x and out start at 16 (bf16: 8) bytes' alignment, four logits
// to an access.
template <bool F32, bool VEC, int SLICE>
__global__ void __launch_bounds__(kThreads)
k_logits_process(LogitsArgs a, int slices) {
    __shared__ __align__(16) uint32_t count[SLICE];
    __shared__ __align__(16) uint32_t bias[SLICE];
    const int64_t row = blockIdx.x / static_cast<uint32_t>(slices);
    const int64_t base = static_cast<int64_t>(blockIdx.x - row * slices) * SLICE;
    const int n = static_cast<int>(a.vocab - base < SLICE ? a.vocab - base : SLICE);
    const int tid = threadIdx.x;
    const bool hist = a.history != nullptr, biased = a.bias_ids != nullptr;
    if (hist || biased) {
        for (int i = 4 * tid; i < SLICE; i += 4 * kThreads) {
            *reinterpret_cast<u32x4*>(count + i) = u32x4{0u, 0u, 0u, 0u};
            *reinterpret_cast<u32x4*>(bias + i) = u32x4{0u, 0u, 0u, 0u};
        }
        __syncthreads();
        if (hist) {
            const int64_t len = min(static_cast<int64_t>(a.history_lens[row]), a.history_stride);
            const int64_t prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
            const int32_t* ids = a.history + row * a.history_stride;
#pragma unroll 4
            for (int64_t i = tid; i < len; i += kThreads) {
                const int64_t t = static_cast<int64_t>(ids[i]) - base;
                if (t < 0 || t >= n) continue;
                if (i < prompt) atomicOr(&count[t], kSeenInPrompt);
                else atomicAdd(&count[t], 1u);
            }
        }
        if (biased) {
            const int64_t len = min(static_cast<int64_t>(a.bias_lens[row]), a.bias_stride);
            const int32_t* ids = a.bias_ids + row * a.bias_stride;
            for (int64_t i = tid; i < len; i += kThreads) {
                const int64_t t = static_cast<int64_t>(ids[i]) - base;
                if (t >= 0 && t < n) atomicMax(&bias[t], static_cast<uint32_t>(i + 1));
            }
        }
        __syncthreads();
    }
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float freq = a.frequency ? a.frequency[row] : 0.0f;
    const float pres = a.presence ? a.presence[row] : 0.0f;
    const uint32_t* mask = nullptr;
    if (a.mask) {
        const int64_t m = a.mask_index ? a.mask_index[row] : row;
        if (m >= 0 && m < a.mask_rows) mask = a.mask + m * a.mask_stride;
    }
    const float* bv = a.bias_values + row * a.bias_stride;
    auto rule = [&](float x, uint32_t cnt, uint32_t bi, bool allowed) {
        if (cnt) x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        const uint32_t times = cnt & ~kSeenInPrompt;
        if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(times))), pres);
        if (bi) x = __fadd_rn(x, bv[bi - 1]);
        return allowed ? x : -INFINITY;
    };
    const int64_t xr = row * a.x_stride + base, orow = row * a.out_stride + base;
    const bool ruled = hist || biased;
    if constexpr (VEC) {
        for (int i = 4 * tid; i < n; i += 4 * kThreads) {
            if (i + 4 <= n) {
                float x[4];
                if constexpr (F32) {
                    const f32x4 v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.x) + xr + i);
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = v[k];
                } else {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const bf16_t*>(a.x) + xr + i);
                    x[0] = bf16w_lo(w[0]); x[1] = bf16w_hi(w[0]); x[2] = bf16w_lo(w[1]); x[3] = bf16w_hi(w[1]);
                }
                u32x4 cnt{0u, 0u, 0u, 0u}, bi{0u, 0u, 0u, 0u};
                if (ruled) {
                    cnt = *reinterpret_cast<const u32x4*>(count + i);
                    bi = *reinterpret_cast<const u32x4*>(bias + i);
                }
                const uint32_t bits = mask ? mask[(base + i) >> 5] >> (i & 31) : 15u;
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = rule(x[k], cnt[k], bi[k], (bits >> k) & 1u);
                if constexpr (F32)
                    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + orow + i) = f32x4{x[0], x[1], x[2], x[3]};
                else
                    *reinterpret_cast<u32x2*>(static_cast<bf16_t*>(a.out) + orow + i) =
                        u32x2{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
            } else {
                for (int k = i; k < n; ++k)
                    store1<F32>(a.out, orow + k,
                                rule(load1<F32>(a.x, xr + k), ruled ? count[k] : 0u, ruled ? bias[k] : 0u,
                                     !mask || ((mask[(base + k) >> 5] >> (k & 31)) & 1u)));
            }
        }
    } else {
        for (int k = tid; k < n; k += kThreads)
            store1<F32>(a.out, orow + k,
                        rule(load1<F32>(a.x, xr + k), ruled ? count[k] : 0u, ruled ? bias[k] : 0u,
                             !mask || ((mask[(base + k) >> 5] >> (k & 31)) & 1u)));
    }
}

template <bool F32, int SLICE>
hipError_t launch(const LogitsArgs& a, bool vec, hipStream_t s) {
    const int64_t slices = ceil_div(a.vocab, SLICE), blocks = a.rows * slices;
    if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(blocks)), block(kThreads);
    if (vec) hipLaunchKernelGGL((k_logits_process<F32, true, SLICE>), grid, block, 0, s, a, static_cast<int>(slices));
    else hipLaunchKernelGGL((k_logits_process<F32, false, SLICE>), grid, block, 0, s, a, static_cast<int>(slices));
    return hipGetLastError();
}

}  // namespace

hipError_t launch_logits_process(const LogitsArgs& a, bool f32, hipStream_t s) {
    if (a.rows <= 0 || a.vocab <= 0) return hipSuccess;
    const uintptr_t mis = (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out)) & (f32 ? 15u : 7u);
    const bool vec = mis == 0 && a.x_stride % 4 == 0 && a.out_stride % 4 == 0;
    return f32 ? launch<true, 4096>(a, vec, s) : launch<false, 4096>(a, vec, s);
}

}  // namespace aps
