// Log probabilities of given tokens, entropies and the likeliest tokens of rows
// of logits (aps_token_logprobs), in one pass over the logits but where many of
// them tie for the likeliest.
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
// LDS and each finds its rank by counting.  Where more than kMost reach it they are
// found one after the other, a pass over the slice each: many equal logits, or a
// mask of a finite value that leaves fewer than `top` groups a token (250 x 100003
// bf16 with 20 tokens a row left, top 20: 507 us beside 34 with a mask of -inf,
// of which no more than `top` are kept).  Logits are ordered by value, then by
// the lower id: a 64-bit key, so the order in which they are collected changes
// nothing.  A row of one slice ends there; others leave maxima, sums and their
// `top` keys in the workspace, and a second launch joins a row's slices in the
// same way.
//
// Bound by the logits' bytes where workgroups are small enough that some load
// while others compute (4096 x 32064 fp32: 178 us with one of 1024 threads on a
// CU, 95 with four slices of 256: 6.1 TB/s in the first launch).
#include <algorithm>

#include "serve.hpp"

namespace aps {
namespace {

constexpr int kMost = 1024;   // keys collected in LDS
constexpr int kGroups = 64;   // and the largest `top`
constexpr int kMaxSlices = 32;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
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
// (+0 for -0, and -inf for a NaN, whose row's sums are NaN)
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
__device__ inline Sums join(int n, Get get, float m = -INFINITY) {
    Sums all = {m, 0.0f, 0.0f};
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
        a.top_logprobs[row * a.top + j] = key_value(top[j]) - o.m - o.log_s;
    }
}

// The `top` largest of `n` keys in LDS into best[0 ..], largest first.
__device__ inline void rank(const u64* keys, int n, u64* best, int top, int tid, int threads) {
    for (int i = tid; i < n; i += threads) {
        const u64 mine = keys[i];
        int above = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) above += keys[j] > mine;
        if (above < top) best[above] = mine;
    }
}

// T threads with N accesses of 16 bytes each; ends of a row that are not on 16
// bytes are at most 2 (U - 1) values, one for each of as many threads of the
// first slice.
template <bool F32, int T, int N>
__global__ void __launch_bounds__(T) k_logprobs(LogprobArgs a, int slices) {
    constexpr int U = F32 ? 4 : 8, WAVES = T / kWave, SPAN = T / kGroups, kSize = F32 ? 4 : 2;
    __shared__ Sums part[WAVES];
    __shared__ __align__(16) float group[kGroups];
    __shared__ float floor_value;
    __shared__ u64 keys[kMost], best[kGroups];
    __shared__ uint16_t hit[T * N];
    __shared__ int count, hits;
    const int64_t row = blockIdx.x / slices;
    const int slice = static_cast<int>(blockIdx.x - row * slices), tid = threadIdx.x, top = a.top;
    const char* x = static_cast<const char*>(a.x) + row * a.x_stride * kSize;
    const int off = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / kSize;
    const int vocab = static_cast<int>(a.vocab), head = off < vocab ? off : vocab;
    const int body = (vocab - head) / U, tail = vocab - head - body * U;   // whole accesses, and what is behind them
    const int v0 = slice * T * N + tid;
    const u32x4* in = reinterpret_cast<const u32x4*>(x + static_cast<int64_t>(head) * kSize);
    constexpr uint32_t kNone = F32 ? 0xFF800000u : 0xFF80FF80u;  // -inf
    u32x4 w[N];   // the row's values stay in registers
#pragma unroll
    for (int n = 0; n < N; ++n) {
        w[n] = u32x4{kNone, kNone, kNone, kNone};
        if (v0 + n * T < body) w[n] = in[v0 + n * T];
    }
    float extra = -INFINITY;
    uint32_t extra_id = 0x40000000u;   // past the vocabulary: nothing
    if (slice == 0 && tid < head + tail) {
        extra_id = static_cast<uint32_t>(tid < head ? tid : vocab - tail + (tid - head));
        extra = load1<F32>(x, extra_id);
    }
    if (tid == 0) count = hits = 0;
    if (tid < top) best[tid] = 0;
    auto value = [&](int n, int u) {
        if constexpr (F32) return __uint_as_float(w[n][u]);
        else return (u & 1) ? bf16w_hi(w[n][u / 2]) : bf16w_lo(w[n][u / 2]);
    };
    // a phase takes the values from their words again rather than hold both
    auto phase = [&]() {
        if constexpr (!F32) {
#pragma unroll
            for (int n = 0; n < N; ++n) asm("" : "+v"(w[n]));
        }
    };
    // the largest number of the thread and of the wave (a NaN is none)
    float mine = fmaxf(extra, -INFINITY);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int u = 0; u < U; ++u) mine = fmaxf(mine, value(n, u));
    float m = mine;
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) {
        if (by == SPAN && top > 1 && tid % SPAN == 0) group[tid / SPAN] = m;
        m = fmaxf(m, __shfl_xor(m, by));
    }
    const float base = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, t = 0.0f;
    auto add = [&](float v) {
        const float d = v - base;                                  // <= 0, -inf, or NaN
        const float e = __builtin_amdgcn_exp2f(d * kLog2e);
        s += e;
        t = fmaf(e, fmaxf(d, -1e4f), t);                           // e is 0 long before (NaN stays in s)
    };
    phase();
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
    if ((tid & 63) == 0) part[tid / kWave] = {m, s, -t};
    __syncthreads();
    const Sums all = join(WAVES, [&](int i) { return part[i]; });
    if (top > 0) {
        if (top > 1) {
            if (tid < kGroups) {
                const float g = group[tid];
                int above = 0, least = 0;
#pragma unroll
                for (int j = 0; j < kGroups; j += 4) {
                    const f32x4 of = *reinterpret_cast<const f32x4*>(group + j);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        above += of[i] > g;
                        least += of[i] >= g;
                    }
                }
                if (above < top && least >= top) floor_value = g;   // equal ones write the same
            }
            __syncthreads();
        }
        const float low = top > 1 ? floor_value : all.m;
        // Fewer than `top` groups with a number: all numbers, and of the others the
        // slice's first `top` ids hold as many as can be wanted.
        const uint32_t window = slice == 0 ? 0u : static_cast<uint32_t>(head + slice * T * N * U);
        auto keep = [&](float v, uint32_t id) {
            v = fmaxf(v, -INFINITY);
            if (!(v >= low) || (low == -INFINITY && v == low && id - window >= static_cast<uint32_t>(top))) return;
            const int at = atomicAdd(&count, 1);
            if (at < kMost) keys[at] = key_of(v, id);
        };
        // the accesses that hold one, then their values: a wave whose every access has
        // some lane's value would else go through all of them
        phase();
        keep(extra, extra_id);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float most = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) most = fmaxf(most, value(n, u));
            if (most >= low && v0 + n * T < body) hit[atomicAdd(&hits, 1)] = static_cast<uint16_t>(n * T + tid);
        }
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < hits; i += T) {
            const int at = slice * T * N + hit[i];
            const u32x4 v = in[at];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if constexpr (F32) keep(__uint_as_float(v[u]), head + at * U + u);
                else keep((u & 1) ? bf16w_hi(v[u / 2]) : bf16w_lo(v[u / 2]), head + at * U + u);
            }
        }
        __syncthreads();
        if (count <= kMost) {
            rank(keys, count, best, top, tid, T);
        } else {
            // too many reach the floor (equal logits, or large ones all in a few
            // groups): one at a time
            u64 last = ~0ull;
#pragma unroll 1
            for (int j = 0; j < top; ++j) {
                u64 k = 0;
                auto next = [&](float v, uint32_t id) {
                    const u64 c = key_of(fmaxf(v, -INFINITY), id);
                    if (c < last) k = max64(k, c);
                };
                next(extra, extra_id);
                const int first = head + slice * T * N * U, end = head + min(body, (slice + 1) * T * N) * U;
#pragma unroll 1
                for (int id = first + tid; id < end; id += T) next(load1<F32>(x, id), id);
#pragma unroll
                for (int by = 1; by < kWave; by *= 2) k = max64(k, shfl_xor64(k, by));
                if ((tid & 63) == 0) keys[tid / kWave] = k;
                __syncthreads();
                k = keys[0];
                for (int i = 1; i < WAVES; ++i) k = max64(k, keys[i]);
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
        u64* to = reinterpret_cast<u64*>(a.part + 4 * a.rows * slices) + at * top;
        for (int j = tid; j < top; j += T) to[j] = best[j];
    }
}

// A wave to a row; what it reads is on its way before anything waits.
template <bool F32>
__global__ void __launch_bounds__(kWave) k_logprobs_join(LogprobArgs a, int slices) {
    __shared__ u64 keys[kMaxSlices * kGroups], best[kGroups];
    __shared__ int count;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    Sums p = {-INFINITY, 0.0f, 0.0f};
    if (tid < slices) {
        const float* part = a.part + 4 * (row * slices + tid);
        p = {part[0], part[1], part[2]};
    }
    const u64* from = reinterpret_cast<const u64*>(a.part + 4 * a.rows * slices) + row * slices * a.top;
    // `top` keys at least reach the largest of the slices' last ones
    u64 floor_key = a.top > 0 && tid < slices ? from[tid * a.top + a.top - 1] : 0;
    if (tid == 0) count = 0;
    if (tid < a.top) best[tid] = 0;
    Sums all = {p.m, 0.0f, 0.0f};
#pragma unroll
    for (int by = 1; by < kMaxSlices; by *= 2) {
        all.m = fmaxf(all.m, __shfl_xor(all.m, by));
        floor_key = max64(floor_key, shfl_xor64(floor_key, by));
    }
    if (tid < slices) {
        const Sums one = join(1, [&](int) { return p; }, all.m);
        all.s = one.s;
        all.w = one.w;
    }
#pragma unroll
    for (int by = 1; by < kMaxSlices; by *= 2) {
        all.s += __shfl_xor(all.s, by);
        all.w += __shfl_xor(all.w, by);
    }
    // (slices are in the first 32 lanes: the others have their own)
    all = {__shfl(all.m, 0), __shfl(all.s, 0), __shfl(all.w, 0)};
    floor_key = static_cast<u64>(__shfl(static_cast<long long>(floor_key), 0));
    __syncthreads();
    if (a.top > 0) {
        for (int i = tid; i < slices * a.top; i += kWave) {
            const u64 k = from[i];
            if (k >= floor_key) keys[atomicAdd(&count, 1)] = k;
        }
        __syncthreads();
        rank(keys, count, best, a.top, tid, kWave);
        __syncthreads();
    }
    write_row<F32>(a, row, all, best, tid, kWave);
}

// The slices of a row: T threads hold kN accesses of 16 bytes.  256 threads, where
// some load while others compute and nothing waits for the slowest of 16 waves, but
// 1024 while no CU has two rows and that spares a row its second launch.  Rows of
// 32064 fp32 in us, 1024 threads and 256: one row 8.4 and 8.7, 256 rows 10.7 and 13.6,
// 300 rows 18.0 and 14.4; bf16, which need half as many slices: one row of 32064 11.0
// and 9.5, 256 rows 12.4 and 12.3, 256 of 50000 13.4 and 17.6.  A row in one slice of
// 256 threads takes 5.8 where 1024 take 8.1.  With 4, 8 and 12 accesses a thread of 256:
// 4096 x 32064 fp32 102, 97, 96; 1000 x 32064 bf16 25, 24, 30; 250 x 100003 bf16, top
// 20, 38, 28, 26.
struct Plan {
    int threads, slices;
};
constexpr int kN = 8;
constexpr int64_t kCus = 256;
Plan plan_of(int64_t rows, int64_t vocab, bool f32) {
    const int64_t accesses = vocab / (f32 ? 4 : 8);
    auto slices = [&](int t) { return static_cast<int>(accesses > 0 ? ceil_div(accesses, int64_t(t) * kN) : 1); };
    const bool one = rows <= kCus && slices(256) > (f32 ? 1 : 2) && slices(1024) == 1;
    if (one || slices(256) > kMaxSlices) return {1024, slices(1024)};
    return {256, slices(256)};
}

template <bool F32, int T>
void slice(const LogprobArgs& a, int slices, hipStream_t s) {
    hipLaunchKernelGGL((k_logprobs<F32, T, kN>), dim3(static_cast<unsigned>(a.rows * slices)), dim3(T), 0, s, a, slices);
}

template <bool F32>
hipError_t run(const LogprobArgs& a, Plan p, hipStream_t s) {
    if (p.threads == 1024) slice<F32, 1024>(a, p.slices, s);
    else slice<F32, 256>(a, p.slices, s);
    if (p.slices > 1)
        hipLaunchKernelGGL(k_logprobs_join<F32>, dim3(static_cast<unsigned>(a.rows)), dim3(kWave), 0, s, a, p.slices);
    return hipGetLastError();
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
    const int64_t most = most_blocks(p.threads) / p.slices;
    for (int64_t first = 0; first < a.rows; first += most) {   // the workspace serves one launch's rows after the other's
        LogprobArgs part = a;
        part.rows = std::min(most, a.rows - first);
        part.x = static_cast<const char*>(a.x) + first * a.x_stride * (f32 ? 4 : 2);
        if (a.n_tokens > 0) part.tokens = a.tokens + first * a.n_tokens, part.logprobs = a.logprobs + first * a.n_tokens;
        if (a.entropy) part.entropy = a.entropy + first;
        if (a.top > 0) part.top_ids = a.top_ids + first * a.top, part.top_logprobs = a.top_logprobs + first * a.top;
        if (const hipError_t e = f32 ? run<true>(part, p, s) : run<false>(part, p, s); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace aps
