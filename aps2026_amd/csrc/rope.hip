// Rotary positions from frequencies: aps_rope turns the first rotary_dim values
// of every head of q and k, aps_rope_table fills the tables that the cache's
// append takes.
//
// The pair i of a row at position p turns by the angle p freq[i]:
//   y0 = A (x0 cos - x1 sin), y1 = A (x0 sin + x1 cos).
// The angle is taken in turns, p (freq / 2 pi), and brought to an eighth of a
// turn around a quarter in 64 bits, where a position past 2^20 still leaves 2^-33
// of a turn; what is left is rounded to fp32 (2^-28 of a turn) and its sine and
// cosine are Taylor's polynomials, whose remainders at pi / 4 are below 2^-28.
// Products and sums are fp32: results are off by about 2^-23 of the pair's norm.
//
// Bound by the bytes of q and k.  A thread computes the angles of its V pairs
// once and turns them in one or two heads of the row, 16 bytes of each half at a
// time, so the trigonometry (some 30 instructions a pair) hides behind the loads.
// 65536 bf16 rows of 20 heads of 128 take 116 us (5.8 TB/s; a large copy has
// 4.9), 8192 rows of which half of each head turns 15.3, one row 3.0.
// Where a start, a stride or a part of a head is off 16 bytes a thread moves one
// value at a time and turns one pair in one or two heads, so that neither the
// accesses nor the angles are hidden: 8192 bf16 rows of 20 heads of 128 34.9 us
// (2.4 TB/s; on 16 bytes 15.7), heads of 80 of which 20 turn 25.0 (2.1 TB/s), fp32
// heads of 128 33.8 (5.0 TB/s).
#include <algorithm>

#include "serve.hpp"

namespace aps {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kCus = 256;
constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A sin and A cos of `turns` of a whole turn.
__device__ inline void sin_cos_turns(double turns, float amplitude, float& s, float& c) {
    const double quarters = 4.0 * (turns - rint(turns));       // [-2, 2]
    const double q = rint(quarters);
    const float x = static_cast<float>(quarters - q) * 1.57079632679489662f;  // [-pi/4, pi/4]
    const float z = x * x;
    float ps = fmaf(z, 2.7557319223985893e-6f, -1.9841269841269841e-4f);      // 1/9!, -1/7!
    ps = fmaf(z, ps, 8.3333333333333333e-3f);
    ps = fmaf(z, ps, -0.16666666666666667f);
    ps = fmaf(x * z, ps, x);
    float pc = fmaf(z, -2.7557319223985888e-7f, 2.4801587301587302e-5f);      // -1/10!, 1/8!
    pc = fmaf(z, pc, -1.3888888888888889e-3f);
    pc = fmaf(z, pc, 4.1666666666666667e-2f);
    pc = fmaf(z, pc, -0.5f);
    pc = fmaf(z, pc, 1.0f);
    const int k = static_cast<int>(q);                                         // quarters: -2 .. 2
    const float a = (k & 1) ? pc : ps, b = (k & 1) ? ps : pc;
    s = amplitude * ((k & 2) ? -a : a);
    c = amplitude * (((k + 1) & 2) ? -b : b);
}

template <bool F32, int V>
__device__ inline void load(const void* base, int64_t at, float (&x)[V]) {
    if constexpr (F32) {
        const float* p = static_cast<const float*>(base) + at;
        if constexpr (V == 4) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
        } else {
            x[0] = p[0];
        }
    } else {
        const bf16_t* p = static_cast<const bf16_t*>(base) + at;
        if constexpr (V == 8) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[2 * i] = bf16w_lo(w[i]); x[2 * i + 1] = bf16w_hi(w[i]); }
        } else {
            x[0] = __uint_as_float(static_cast<uint32_t>(p[0]) << 16);
        }
    }
}

template <bool F32, int V>
__device__ inline void store(void* base, int64_t at, const float (&x)[V]) {
    if constexpr (F32) {
        float* p = static_cast<float*>(base) + at;
        if constexpr (V == 4) {
            *reinterpret_cast<u32x4*>(p) = u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                                                 __float_as_uint(x[3])};
        } else {
            p[0] = x[0];
        }
    } else {
        bf16_t* p = static_cast<bf16_t*>(base) + at;
        if constexpr (V == 8) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack2_bf16(x[2 * i], x[2 * i + 1]);
            *reinterpret_cast<u32x4*>(p) = w;
        } else {
            p[0] = static_cast<bf16_t>(pack2_bf16(x[0], 0.0f) & 0xFFFFu);
        }
    }
}

// V values (16 bytes, or 1) to an access.  A row has `turning` threads' worth of
// pairs, V each, and `still` of 2 V values behind them that are only copied;
// `spread` threads share the heads of one such place.
struct Shape {
    int turning, still, spread, rows_a_block;
};

template <bool F32, int V, bool PAIRS>
__global__ void __launch_bounds__(kThreads) k_rope(RopeArgs a, Shape p) {
    const int places = p.turning + p.still, per_row = places * p.spread;
    const int half = a.rotary_dim / 2, heads = a.q_heads + a.k_heads;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * p.rows_a_block;
    for (int item = threadIdx.x; item < per_row * p.rows_a_block; item += kThreads) {
        const int r = item / per_row, rest = item - r * per_row;
        const int share = rest / places, place = rest - share * places;
        const int64_t row = first + r;
        if (row >= a.rows) return;
        const int64_t pos = a.positions[row];
        const bool turns = place < p.turning && pos >= 0;
        // this thread's two runs of V values in a head, and how much of the second is there
        int at0, at1;
        if (place < p.turning) {
            at0 = PAIRS ? 2 * V * place : V * place;
            at1 = at0 + (PAIRS ? V : half);
        } else {
            at0 = a.rotary_dim + 2 * V * (place - p.turning);
            at1 = at0 + V;
        }
        const bool second = at1 < a.head_dim;
        float s[V], c[V];
        if (turns) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                sin_cos_turns(static_cast<double>(pos) * (a.freq[V * place + i] * kTurn), a.amplitude, s[i], c[i]);
                if (a.inverse) s[i] = -s[i];
            }
        }
        for (int h = share; h < heads; h += p.spread) {
            const bool is_q = h < a.q_heads;
            const int64_t head = static_cast<int64_t>(is_q ? h : h - a.q_heads) * a.head_dim;
            const void* from = is_q ? a.q : a.k;
            void* to = is_q ? a.q_out : a.k_out;
            const int64_t in = row * (is_q ? a.q_stride : a.k_stride) + head;
            const int64_t out = row * (is_q ? a.q_out_stride : a.k_out_stride) + head;
            float x0[V], x1[V];
            load<F32, V>(from, in + at0, x0);
            if (second) load<F32, V>(from, in + at1, x1);
            if (turns) {
                if constexpr (!PAIRS || V == 1) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float u = x0[i], w = x1[i];
                        x0[i] = fmaf(u, c[i], -(w * s[i]));
                        x1[i] = fmaf(u, s[i], w * c[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V / 2; ++i) {
                        float u = x0[2 * i], w = x0[2 * i + 1];
                        x0[2 * i] = fmaf(u, c[i], -(w * s[i]));
                        x0[2 * i + 1] = fmaf(u, s[i], w * c[i]);
                        u = x1[2 * i], w = x1[2 * i + 1];
                        x1[2 * i] = fmaf(u, c[V / 2 + i], -(w * s[V / 2 + i]));
                        x1[2 * i + 1] = fmaf(u, s[V / 2 + i], w * c[V / 2 + i]);
                    }
                }
            }
            store<F32, V>(to, out + at0, x0);
            if (second) store<F32, V>(to, out + at1, x1);
        }
    }
}

// A thread to an angle: bound by the bytes of the tables (1048576 positions of 64
// pairs 129 us, 4.2 TB/s; 4096 positions 8.2, a launch and two tensors).
__global__ void __launch_bounds__(kThreads)
k_rope_table(const double* __restrict__ freq, int pairs, int64_t first, int64_t count, float amplitude, float* cosv,
             float* sinv) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= count * pairs) return;
    const int64_t row = i / pairs;
    sin_cos_turns(static_cast<double>(first + row) * (freq[i - row * pairs] * kTurn), amplitude, sinv[i], cosv[i]);
}

template <bool F32, int V>
hipError_t launch(const RopeArgs& a, hipStream_t s) {
    Shape p;
    p.turning = a.rotary_dim / 2 / V;
    p.still = static_cast<int>(ceil_div(a.head_dim - a.rotary_dim, 2 * V));
    const int heads = a.q_heads + a.k_heads, places = p.turning + p.still;
    p.spread = heads;
    p.rows_a_block = static_cast<int>(kThreads / (places * p.spread));
    // Two heads a thread where one would give every CU a workgroup and more: 65536 rows
    // 145 us with one, 116 with two (three 116, four 121), 8192 rows 21 and 15.7; 512
    // rows 4.4 either way, 64 rows 3.75 with one and 4.1 with two.
    if (a.rows > kCus * std::max(p.rows_a_block, 1)) {
        p.spread = static_cast<int>(ceil_div(heads, 2));
        p.rows_a_block = static_cast<int>(kThreads / (places * p.spread));
    }
    if (p.rows_a_block < 1) p.rows_a_block = 1;
    const int64_t most = most_blocks(kThreads) * p.rows_a_block;
    for (int64_t first = 0; first < a.rows; first += most) {
        constexpr int64_t kSize = F32 ? 4 : 2;
        RopeArgs part = a;
        part.rows = std::min(most, a.rows - first);
        part.positions += first;
        part.q = static_cast<const char*>(a.q) + first * a.q_stride * kSize;
        part.q_out = static_cast<char*>(a.q_out) + first * a.q_out_stride * kSize;
        if (a.k_heads > 0) {
            part.k = static_cast<const char*>(a.k) + first * a.k_stride * kSize;
            part.k_out = static_cast<char*>(a.k_out) + first * a.k_out_stride * kSize;
        }
        const dim3 grid(static_cast<unsigned>(ceil_div(part.rows, p.rows_a_block)));
        if (a.pairs) hipLaunchKernelGGL((k_rope<F32, V, true>), grid, dim3(kThreads), 0, s, part, p);
        else hipLaunchKernelGGL((k_rope<F32, V, false>), grid, dim3(kThreads), 0, s, part, p);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, bool f32, hipStream_t s) {
    if (a.rows <= 0 || a.q_heads + a.k_heads <= 0) return hipSuccess;
    const int v = f32 ? 4 : 8;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) |
                         reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.k_out);
    // 16-byte accesses where every run of v values starts at 16 bytes
    const bool vec = (at & 15u) == 0 && a.head_dim % v == 0 && a.rotary_dim / 2 % v == 0 && a.q_stride % v == 0 &&
                     a.q_out_stride % v == 0 && a.k_stride % v == 0 && a.k_out_stride % v == 0;
    if (f32) return vec ? launch<true, 4>(a, s) : launch<true, 1>(a, s);
    return vec ? launch<false, 8>(a, s) : launch<false, 1>(a, s);
}

hipError_t launch_rope_table(const double* freq, int pairs, int64_t first, int64_t count, float amplitude,
                             float* cosv, float* sinv, hipStream_t s) {
    if (count <= 0 || pairs <= 0) return hipSuccess;
    const int64_t most = most_blocks(kThreads) * kThreads / pairs;   // positions of a launch
    for (int64_t at = 0; at < count; at += most) {
        const int64_t n = std::min(most, count - at);
        const dim3 grid(static_cast<unsigned>(ceil_div(n * pairs, kThreads)));
        hipLaunchKernelGGL(k_rope_table, grid, dim3(kThreads), 0, s, freq, pairs, first + at, n, amplitude,
                           cosv + at * pairs, sinv + at * pairs);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace aps
