// Log probabilities of given tokens, entropies and the likeliest tokens of rows
// of logits (aps_token_logprobs), in one pass over the logits.
//
//   m = max x, S = sum exp(x - m), W = sum exp(x - m) (m - x)
//   log p(t) = (x[t] - m) - log S,  entropy = log S + W / S
// W's terms are all positive and its factor is the distance that the exponent
// has too, so nothing cancels.
//
// A workgroup holds a slice of a row in registers.  Each wave takes its own
// maximum and sums, which are then joined by
//   m = max m_i, S = sum S_i e^(m_i - m), W = sum e^(m_i - m) (W_i + S_i (m - m_i)).
// The likeliest `top` need no sort of the row: the slice's threads form 64
// groups, and the top-th largest of the groups' largest logits is a floor that
// `top` logits at least reach.  Those that reach it (some tens) are collected in
// LDS and each finds its rank by counting.  Logits are ordered by value, then by
// the lower id: a 64-bit key, so the order in which they are collected changes
// nothing.  A row of one slice ends there; others leave maxima, sums and their
// `top` keys in the workspace, and a second launch joins a row's slices in the
// same way.
#include "serve.hpp"

namespace aps {
namespace {

constexpr int kMost = 1024;   // keys collected in LDS
constexpr int kGroups = 64;   // and the largest `top`
constexpr int kMaxSlices = 32;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

template <bool F32>
__device__ inline float load1(const void* p, int64_t i) {
    if constexpr (F32) return static_cast<const float*>(p)[i];
    else return __uint_as_float(static_cast<uint32_t>(static_cast<const bf16_t*>(p)[i]) << 16);
}

// Larger for the larger value, then for the lower id; +0 and -0 are equal.
__device__ inline u64 key_of(float x, uint32_t id) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t up = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return static_cast<u64>(up) << 32 | (0xFFFFFFFFu - id);
}
__device__ inline float key_value(u64 key) {
    const uint32_t up = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(up & 0x80000000u ? up ^ 0x80000000u : ~up);
}
__device__ inline uint32_t key_id(u64 key) { return 0xFFFFFFFFu - static_cast<uint32_t>(key); }

__device__ inline u64 max64(u64 a, u64 b) { return a > b ? a : b; }
__device__ inline u64 shfl_xor64(u64 v, int by) { return static_cast<u64>(__shfl_xor(static_cast<long long>(v), by)); }

struct Sums { float m, s, w; };

// e^(from - to) for from <= to, 0 from -inf.
__device__ inline float shrink(float from, float to) {
    return from == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((from - to) * kLog2e);
}
template <typename Get>
__device__ inline Sums join(int n, Get get) {
    Sums all = {-INFINITY, 0.0f, 0.0f};
    for (int i = 0; i < n; ++i) all.m = fmaxf(all.m, get(i).m);
    for (int i = 0; i < n; ++i) {
        const Sums p = get(i);
        const float f = shrink(p.m, all.m);
        const float d = p.m == -INFINITY ? 0.0f : fminf(all.m - p.m, 1e4f);  // f is 0 long before
        all.s += f * p.s;
        all.w += f * fmaf(p.s, d, p.w);
    }
    return all;
}

struct Out {
    float log_s, m, entropy;
};
// A row with nothing above -inf has no distribution: log p = -inf, entropy 0.
__device__ inline Out finish(Sums t) {
    if (t.m == -INFINITY && t.s == 0.0f) return {0.0f, 0.0f, 0.0f};
    const float l = logf(t.s);
    return {l, t.m, l + t.w / t.s};
}

template <bool F32>
__device__ inline void write_row(const LogprobArgs& a, int64_t row, Sums t, const u64* top, int tid, int threads) {
    const Out o = finish(t);
    if (tid == 0 && a.entropy) a.entropy[row] = o.entropy;
    for (int64_t j = tid; j < a.n_tokens; j += threads) {
        const int64_t id = a.tokens[row * a.n_tokens + j];
        a.logprobs[row * a.n_tokens + j] =
            id < 0 || id >= a.vocab ? 0.0f : load1<F32>(a.x, row * a.x_stride + id) - o.m - o.log_s;
    }
    for (int j = tid; j < a.top; j += threads) {
        a.top_ids[row * a.top + j] = static_cast<int32_t>(key_id(top[j]));
        a.top_logprobs[row * a.top + j] = load1<F32>(a.x, row * a.x_stride + key_id(top[j])) - o.m - o.log_s;
    }
}

// The `top` largest of `n` keys in LDS into best[0 ..], largest first.
__device__ inline void rank(const u64* keys, int n, u64* best, int top, int tid, int threads) {
    for (int i = tid; i < n; i += threads) {
        const u64 mine = keys[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += keys[j] > mine;
        if (above < top) best[above] = mine;
    }
}

// T threads with N accesses of 16 bytes each; ends of a row that are not on 16
// bytes are at most 2 (U - 1) values, one for each of as many threads of the
// first slice.
template <bool F32, int T, int N>
__global__ void __launch_bounds__(T) k_logprobs(LogprobArgs a, int slices) {
    constexpr int U = F32 ? 4 : 8, WAVES = T / kWave, SPAN = T / kGroups;
    __shared__ Sums part[WAVES];
    __shared__ u64 group[kGroups], keys[kMost], best[kGroups], floor_key;
    __shared__ int count;
    const int64_t row = blockIdx.x / slices;
    const int slice = static_cast<int>(blockIdx.x - row * slices), tid = threadIdx.x;
    const char* x = static_cast<const char*>(a.x) + row * a.x_stride * (F32 ? 4 : 2);
    constexpr int kSize = F32 ? 4 : 2;
    const int off = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / kSize;
    const int head = off < a.vocab ? off : static_cast<int>(a.vocab);
    const int vocab = static_cast<int>(a.vocab), body = (vocab - head) / U;  // whole accesses
    const int tail = vocab - head - body * U;
    const int v0 = slice * T * N + tid;
    const u32x4* in = reinterpret_cast<const u32x4*>(x + static_cast<int64_t>(head) * kSize);
    constexpr uint32_t kNone = F32 ? 0xFF800000u : 0xFF80FF80u;  // -inf
    u32x4 w[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int v = v0 + n * T;
        w[n] = u32x4{kNone, kNone, kNone, kNone};
        if (v < body) w[n] = in[v];
    }
    float extra = -INFINITY;
    uint32_t extra_id = 0x40000000u + tid;  // ids past the vocabulary stand for nothing
    if (slice == 0 && tid < head + tail) {
        extra_id = static_cast<uint32_t>(tid < head ? tid : vocab - tail + (tid - head));
        extra = load1<F32>(x, extra_id);
    }
    auto value = [&](int n, int u) {
        if constexpr (F32) return __uint_as_float(w[n][u]);
        else return (u & 1) ? bf16w_hi(w[n][u / 2]) : bf16w_lo(w[n][u / 2]);
    };
    auto id_of = [&](int n, int u) {
        const int v = v0 + n * T;
        return static_cast<uint32_t>(head + v * U + u) + (v < body ? 0u : 0x40000000u);
    };
    // maximum of what is a number, of the thread and of the wave
    float mine = fmaxf(extra, -INFINITY);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int u = 0; u < U; ++u) mine = fmaxf(mine, value(n, u));
    float m = mine;
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) m = fmaxf(m, __shfl_xor(m, by));
    const float base = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, t = 0.0f;
    auto add = [&](float v) {
        const float d = base - v;                       // >= 0, inf for -inf, NaN
        const float e = __builtin_amdgcn_exp2f(d * -kLog2e);
        s += e;
        t = fmaf(e, fminf(d, 1e4f), t);                 // e is 0 long before (NaN stays in s)
    };
    add(extra);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int u = 0; u < U; ++u) add(value(n, u));
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) {
        s += __shfl_xor(s, by);
        t += __shfl_xor(t, by);
    }
    if ((tid & 63) == 0) part[tid / kWave] = {m, s, t};
    if (a.top > 0) {
        // the thread's first largest, then its group's
        uint32_t id = 0x40000000u + extra_id;
#pragma unroll
        for (int n = N - 1; n >= 0; --n)
#pragma unroll
            for (int u = U - 1; u >= 0; --u) {
                if (fmaxf(value(n, u), -INFINITY) == mine) id = id_of(n, u);
            }
        if (fmaxf(extra, -INFINITY) == mine && extra_id < id) id = extra_id;
        u64 k = key_of(mine, id);
#pragma unroll
        for (int by = 1; by < SPAN; by *= 2) k = max64(k, shfl_xor64(k, by));
        if (tid % SPAN == 0) group[tid / SPAN] = k;
        if (tid == 0) count = 0;
    }
    __syncthreads();
    const Sums all = join(WAVES, [&](int i) { return part[i]; });
    if (a.top == 1) {
        if (tid < kGroups) {
            u64 k = group[tid];
#pragma unroll
            for (int by = 1; by < kWave; by *= 2) k = max64(k, shfl_xor64(k, by));
            if (tid == 0) best[0] = k;
        }
        __syncthreads();
    } else if (a.top > 1) {
        if (tid < kGroups) {
            const u64 k = group[tid];
            int above = 0;
            for (int j = 0; j < kGroups; ++j) above += group[j] > k;
            if (above == a.top - 1) floor_key = k;
        }
        __syncthreads();
        const u64 least = floor_key;
        const float low = key_value(least);
        auto keep = [&](float v, uint32_t id) {
            v = fmaxf(v, -INFINITY);
            if (v < low) return;
            const u64 k = key_of(v, id);
            if (k < least) return;
            const int at = atomicAdd(&count, 1);
            if (at < kMost) keys[at] = k;
        };
        keep(extra, extra_id);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                keep(value(n, u), id_of(n, u));
            }
        __syncthreads();
        if (count <= kMost) {
            rank(keys, count, best, a.top, tid, T);
        } else {
            // too many reach the floor (large logits all in a few groups): one at a time
            u64 last = ~0ull;
            for (int j = 0; j < a.top; ++j) {
                u64 k = 0;
                auto next = [&](float v, uint32_t id) {
                    const u64 c = key_of(fmaxf(v, -INFINITY), id);
                    if (c < last) k = max64(k, c);
                };
                next(extra, extra_id);
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                                next(value(n, u), id_of(n, u));
                    }
#pragma unroll
                for (int by = 1; by < kWave; by *= 2) k = max64(k, shfl_xor64(k, by));
                if ((tid & 63) == 0) group[tid / kWave] = k;
                __syncthreads();
                k = group[0];
                for (int i = 1; i < WAVES; ++i) k = max64(k, group[i]);
                last = k;
                if (tid == 0) best[j] = k;
                __syncthreads();
            }
        }
        __syncthreads();
    }
    if (slices == 1) {
        write_row<F32>(a, row, all, best, tid, T);
    } else {
        const int64_t at = row * slices + slice;
        if (tid == 0) {
            float* to = a.part + 4 * at;
            to[0] = all.m;
            to[1] = all.s;
            to[2] = all.w;
        }
        u64* to = reinterpret_cast<u64*>(a.part + 4 * a.rows * slices) + at * a.top;
        for (int j = tid; j < a.top; j += T) to[j] = best[j];
    }
}

template <bool F32>
__global__ void __launch_bounds__(256) k_logprobs_join(LogprobArgs a, int slices) {
    __shared__ u64 keys[kMaxSlices * kGroups], best[kGroups], floor_key;
    __shared__ int count;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const float* part = a.part + 4 * row * slices;
    const Sums all = join(slices, [&](int i) { return Sums{part[4 * i], part[4 * i + 1], part[4 * i + 2]}; });
    if (a.top > 0) {
        const u64* from = reinterpret_cast<const u64*>(a.part + 4 * a.rows * slices) + row * slices * a.top;
        // `top` keys at least reach the largest of the slices' last ones
        if (tid == 0) { floor_key = 0; count = 0; }
        __syncthreads();
        for (int i = tid; i < slices; i += 256) atomicMax(&floor_key, from[static_cast<int64_t>(i) * a.top + a.top - 1]);
        __syncthreads();
        for (int i = tid; i < slices * a.top; i += 256) {
            const u64 k = from[i];
            if (k >= floor_key) keys[atomicAdd(&count, 1)] = k;
        }
        __syncthreads();
        rank(keys, count, best, a.top, tid, 256);
        __syncthreads();
    }
    write_row<F32>(a, row, all, best, tid, 256);
}

// The slices of a row: T threads hold N accesses of 16 bytes.
struct Plan {
    int threads, slices;
};
constexpr int kN = 8;
Plan plan_of(int64_t rows, int64_t vocab, bool f32) {
    const int64_t accesses = vocab / (f32 ? 4 : 8);
    auto slices = [&](int t) { return static_cast<int>(accesses > 0 ? ceil_div(accesses, int64_t(t) * kN) : 1); };
    if (slices(1024) == 1 || slices(256) > kMaxSlices) return {1024, slices(1024)};
    return {256, slices(256)};
}

template <bool F32, int T>
void slice(const LogprobArgs& a, int slices, hipStream_t s) {
    hipLaunchKernelGGL((k_logprobs<F32, T, kN>), dim3(static_cast<unsigned>(a.rows * slices)), dim3(T), 0, s, a, slices);
}

}  // namespace

int64_t token_logprobs_blocks(int64_t rows, int64_t vocab, bool f32) { return rows * plan_of(rows, vocab, f32).slices; }

size_t token_logprobs_part_bytes(int64_t rows, int64_t vocab, int top, bool f32) {
    const Plan p = plan_of(rows, vocab, f32);
    return p.slices == 1 ? 0 : static_cast<size_t>(rows) * p.slices * (16 + 8 * static_cast<size_t>(top));
}

hipError_t launch_token_logprobs(const LogprobArgs& a, bool f32, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    const Plan p = plan_of(a.rows, a.vocab, f32);
    if (f32) {
        if (p.threads == 1024) slice<true, 1024>(a, p.slices, s);
        else slice<true, 256>(a, p.slices, s);
    } else {
        if (p.threads == 1024) slice<false, 1024>(a, p.slices, s);
        else slice<false, 256>(a, p.slices, s);
    }
    if (p.slices > 1) {
        const dim3 grid(static_cast<unsigned>(a.rows));
        if (f32) hipLaunchKernelGGL(k_logprobs_join<true>, grid, dim3(256), 0, s, a, p.slices);
        else hipLaunchKernelGGL(k_logprobs_join<false>, grid, dim3(256), 0, s, a, p.slices);
    }
    return hipGetLastError();
}

}  // namespace aps
