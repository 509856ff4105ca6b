// Linear layers with weights in 4 bits (aps_linear_q4): y = x W^T + b with
// W[n][k] = (code - zero) scale, a scale and a zero for each `group` inputs; and
// aps_quantise_q4, which makes such weights.
//
// The matrix cores do the products for one row as for many: they take the codes
// with the fewest instructions.  A code c becomes the bf16 value 1 + c / 16 by
// putting its bits below an exponent (a shift and an and-or for two), and
//   sum_k x (c - zero) scale = 16 scale (sum_k x (1 + c / 16) - (1 + zero / 16) sum_k x)
// over each group, where sum_k x is the product with a matrix of ones, which lies
// in the accumulators as the other sum does.  All products are exact, sums are
// fp32.  An offset of 16 + zero codes, not the 128 of codes in the lowest bits,
// costs the fp32 sums 2 to 3 bits of a group's own sum: about 3e-7 of y where
// an fp32 chain over the inputs has 5e-7.
//
// fp32 x is the sum of three bf16 terms (8 bits each, cut off one after the
// other), so its products are exact too.  Up to five rows have their terms side
// by side as rows of the matrix cores' 16; for more rows a launch before writes
// the terms to the workspace.
//
// A lane loads 16 bytes, 32 codes of a row; the four lanes of a row hold 128
// neighbouring codes, so four swaps between the lanes' quarters (a 4 x 4
// transpose of words) give every product step 32 neighbouring inputs, the
// smallest group.  Within a lane's word of 8 codes the pairs of a register are
// (i, i + 4); x is put in the same order.
//
// A workgroup's waves share its columns and take the 256-input pieces (a 128-byte
// line of every row) in turn; their sums are joined in LDS in a fixed order.
// Bound by the codes' bytes up to some 64 rows.
#include "serve.hpp"

namespace aps {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kPiece = 256;      // inputs of a wave's turn: two loads of codes
constexpr int kPackRows = 5;     // fp32 rows whose three terms fit in 16
constexpr int kTermPitch = 272;  // bytes of a row of 128 terms in LDS

enum class X { kBf16, kPack, kTerms };

__device__ inline bf16x8 frag(u32x4 w) { return __builtin_bit_cast(bf16x8, w); }
__device__ inline f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Register r of the lanes' quarter q <- register q of quarter r.
__device__ inline u32x4 transpose_quarters(u32x4 w) {
    const auto a = __builtin_amdgcn_permlane16_swap(w[0], w[1], false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(w[2], w[3], false, false);
    const auto c = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
    return u32x4{c[0], d[0], c[1], d[1]};
}

// Eight codes as bf16 1 + c / 16: (0, 4), (1, 5), (2, 6), (3, 7).
__device__ inline bf16x8 code_values(uint32_t w) {
    constexpr uint32_t kMask = 0x00780078u, kOne = 0x3F803F80u;
    return frag(u32x4{((w << 3) & kMask) | kOne, ((w >> 1) & kMask) | kOne, ((w >> 5) & kMask) | kOne,
                      ((w >> 9) & kMask) | kOne});
}

// Eight neighbouring bf16 values in the codes' order.
__device__ inline u32x4 code_order(u32x4 w) {
    return u32x4{__builtin_amdgcn_perm(w[2], w[0], 0x05040100u), __builtin_amdgcn_perm(w[2], w[0], 0x07060302u),
                 __builtin_amdgcn_perm(w[3], w[1], 0x05040100u), __builtin_amdgcn_perm(w[3], w[1], 0x07060302u)};
}

// The three bf16 terms of eight fp32 values, in the codes' order.
__device__ inline void terms_of(const float (&x)[8], u32x4 (&t)[3]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            t[j][i] = __builtin_amdgcn_perm(__float_as_uint(v[i + 4]), __float_as_uint(v[i]), 0x07060302u);
        if (j < 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] - __uint_as_float(__float_as_uint(v[i]) & 0xFFFF0000u);
        }
    }
}

__device__ inline void load8(const float* p, bool vec, float (&x)[8]) {
    if (vec) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}
__device__ inline u32x4 load8(const bf16_t* p, bool vec) {
    if (vec) return *reinterpret_cast<const u32x4*>(p);
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = static_cast<uint32_t>(p[2 * i]) | static_cast<uint32_t>(p[2 * i + 1]) << 16;
    return w;
}

// fp32 x [rows][in] -> [3][rows][in] bf16 terms in the codes' order.
__global__ void __launch_bounds__(256)
k_q4_terms(const float* __restrict__ x, int64_t stride, int64_t rows, int in, bool vec, bf16_t* __restrict__ to) {
    const int64_t runs = in / 8, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= rows * runs) return;
    const int64_t row = i / runs, at = (i - row * runs) * 8;
    float v[8];
    u32x4 t[3];
    load8(x + row * stride + at, vec, v);
    terms_of(v, t);
#pragma unroll
    for (int j = 0; j < 3; ++j) *reinterpret_cast<u32x4*>(to + (j * rows + row) * in + at) = t[j];
}

template <int MT, int NT, int GROUP, X KIND, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
k_linear_q4(LinearQ4Args a, bool x_vec, int n_blocks, int m_blocks) {
    constexpr int GROUPS = kPiece / GROUP, STEPS = GROUP / 32;  // of a piece; product steps of a group
    constexpr int TERMS = KIND == X::kTerms ? 3 : 1;
    constexpr int COLS = 16 * NT, RED = WAVES * 16 * MT * COLS * 4;
    constexpr int PACK = KIND == X::kPack ? WAVES * 16 * kTermPitch : 0;
    __shared__ __align__(16) unsigned char lds[RED > PACK ? RED : PACK];
    const int wave = threadIdx.x / 64, lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4;
    // blocks of the same columns on one XCD (workgroups go round the eight)
    int nb = blockIdx.x, mb = 0;
    if (m_blocks > 1) {
        const int turn = blockIdx.x / 8;
        nb = (turn / m_blocks) * 8 + (blockIdx.x & 7);
        mb = turn % m_blocks;
        if (nb >= n_blocks) return;
    }
    const int in = a.w.in, groups = in / GROUP;
    const int64_t m0 = static_cast<int64_t>(mb) * 16 * MT;
    const int n0 = nb * COLS;
    const uint8_t* code_row[NT];
    int64_t scale_row[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int n = min(n0 + 16 * j + col, a.w.out - 1);
        code_row[j] = a.w.codes + static_cast<int64_t>(n) * (in / 2) + 16 * q;
        scale_row[j] = static_cast<int64_t>(n) * groups;
    }
    int64_t x_row[MT];  // of the lane's row of each tile
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = min(m0 + 16 * i + col, a.rows - 1);
        x_row[i] = m * (KIND == X::kTerms ? in : a.x_stride);
    }
    struct Held { u32x4 code[2][NT]; };
    auto fetch = [&](int piece) {
        Held h;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int k = piece * kPiece + 128 * c + 32 * q;
                h.code[c][j] = u32x4{0u, 0u, 0u, 0u};
                if (k < in) h.code[c][j] = *reinterpret_cast<const u32x4*>(code_row[j] + (piece * kPiece + 128 * c) / 2);
            }
        return h;
    };
    const f32x4 zero4 = {0.0f, 0.0f, 0.0f, 0.0f};
    const bf16x8 ones = frag(u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
    f32x4 total[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) total[j][i] = zero4;
    const int pieces = (in + kPiece - 1) / kPiece;
    Held now{};
    if (wave < pieces) now = fetch(wave);
    for (int piece = wave; piece < pieces; piece += WAVES) {
        const int k0 = piece * kPiece;
        // scales and zeros of the piece's groups: 16 scale, -(1 + zero / 16)
        float scale[NT][GROUPS], off[NT][GROUPS];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                scale[j][g] = 0.0f;
                off[j][g] = -1.5f;
                if (k0 + g * GROUP < in) {
                    const int64_t at = scale_row[j] + piece * GROUPS + g;
                    scale[j][g] = a.w.scales_f32
                                      ? static_cast<const float*>(a.w.scales)[at]
                                      : __uint_as_float(static_cast<uint32_t>(static_cast<const bf16_t*>(a.w.scales)[at]) << 16);
                    if (a.w.zeros) off[j][g] = fmaf(static_cast<float>(a.w.zeros[at]), -0.0625f, -1.0f);
                }
            }
        Held next{};
        if (piece + WAVES < pieces) next = fetch(piece + WAVES);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int kc = k0 + 128 * c;
            if (kc >= in) break;
            unsigned char* mine = lds + wave * 16 * kTermPitch;
            if constexpr (KIND == X::kPack) {
                // 16 runs of 8 values a row: their terms into rows 3 m, 3 m + 1, 3 m + 2
                for (int run = lane; run < static_cast<int>(a.rows) * 16; run += 64) {
                    const int m = run >> 4, k = kc + 8 * (run & 15);
                    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                    if (k < in) load8(static_cast<const float*>(a.x) + m * a.x_stride + k, x_vec, v);
                    u32x4 t[3];
                    terms_of(v, t);
#pragma unroll
                    for (int j = 0; j < 3; ++j)
                        *reinterpret_cast<u32x4*>(mine + (3 * m + j) * kTermPitch + 16 * (run & 15)) = t[j];
                }
                __builtin_amdgcn_wave_barrier();
            }
            u32x4 code[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) code[j] = transpose_quarters(now.code[c][j]);
#pragma unroll
            for (int g = 0; g < 128 / GROUP; ++g) {
                f32x4 sum[MT], dot[NT][MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    sum[i] = zero4;
#pragma unroll
                    for (int j = 0; j < NT; ++j) dot[j][i] = zero4;
                }
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    const int t = g * STEPS + s, k = kc + 32 * t;
                    bf16x8 xs[TERMS][MT];
#pragma unroll
                    for (int e = 0; e < TERMS; ++e)
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            u32x4 w = {0u, 0u, 0u, 0u};
                            if constexpr (KIND == X::kPack) {
                                w = *reinterpret_cast<const u32x4*>(mine + col * kTermPitch + 64 * t + 16 * q);
                            } else if (k < in) {
                                if constexpr (KIND == X::kTerms)
                                    w = *reinterpret_cast<const u32x4*>(a.terms + e * a.rows * in + x_row[i] + k + 8 * q);
                                else
                                    w = code_order(load8(static_cast<const bf16_t*>(a.x) + x_row[i] + k + 8 * q, x_vec));
                            }
                            xs[e][i] = frag(w);
                        }
#pragma unroll
                    for (int e = 0; e < TERMS; ++e)
#pragma unroll
                        for (int i = 0; i < MT; ++i) sum[i] = mfma(xs[e][i], ones, sum[i]);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const bf16x8 v = code_values(code[j][t]);
#pragma unroll
                        for (int e = 0; e < TERMS; ++e)
#pragma unroll
                            for (int i = 0; i < MT; ++i) dot[j][i] = mfma(xs[e][i], v, dot[j][i]);
                    }
                }
                const int at = c * (128 / GROUP) + g;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            total[j][i][r] = fmaf(scale[j][at], fmaf(off[j][at], sum[i][r], dot[j][i][r]), total[j][i][r]);
            }
            if constexpr (KIND == X::kPack) __builtin_amdgcn_wave_barrier();
        }
        now = next;
    }
    // join the waves: [wave][row][column]
    __syncthreads();
    float* red = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                red[(wave * 16 * MT + 16 * i + 4 * q + r) * COLS + 16 * j + col] = total[j][i][r];
    __syncthreads();
    const int64_t left = a.rows - m0;
    const int m_rows = left < 16 * MT ? static_cast<int>(left) : 16 * MT;
    for (int e = threadIdx.x; e < m_rows * COLS; e += 64 * WAVES) {
        const int m = e / COLS, n = n0 + e % COLS;
        if (n >= a.w.out) continue;
        float y = 0.0f;
        for (int w = 0; w < WAVES; ++w) {
            if constexpr (KIND == X::kPack) {
#pragma unroll
                for (int t = 2; t >= 0; --t) y += red[(w * 16 + 3 * m + t) * COLS + e % COLS];
            } else {
                y += red[(w * 16 * MT + m) * COLS + e % COLS];
            }
        }
        y *= 16.0f;
        if (a.bias) y += a.bias[n];
        const int64_t to = (m0 + m) * a.w.out + n;
        if constexpr (KIND == X::kBf16) static_cast<bf16_t*>(a.y)[to] = static_cast<bf16_t>(pack2_bf16(y, 0.0f) & 0xFFFFu);
        else static_cast<float*>(a.y)[to] = y;
    }
}

// Eight neighbouring values of a weight's row to a thread, its group's in
// neighbouring lanes.
template <bool F32, bool ZEROS>
__global__ void __launch_bounds__(256)
k_quantise_q4(const void* __restrict__ w, int64_t runs, int lanes, uint32_t* __restrict__ codes, void* scales,
              bool scales_f32, uint8_t* zeros) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const bool live = i < runs;   // whole groups leave together, but the lanes' exchange needs all
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
        if constexpr (F32) {
            load8(static_cast<const float*>(w) + 8 * i, true, x);
        } else {
            const u32x4 v = load8(static_cast<const bf16_t*>(w) + 8 * i, true);
#pragma unroll
            for (int k = 0; k < 4; ++k) { x[2 * k] = bf16w_lo(v[k]); x[2 * k + 1] = bf16w_hi(v[k]); }
        }
    }
    float lo = 0.0f, hi = 0.0f;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        lo = fminf(lo, x[k]);
        hi = fmaxf(hi, x[k]);
        bad |= !(x[k] - x[k] == 0.0f);
    }
    for (int by = 1; by < lanes; by *= 2) {
        lo = fminf(lo, __shfl_xor(lo, by));
        hi = fmaxf(hi, __shfl_xor(hi, by));
        bad |= __shfl_xor(static_cast<int>(bad), by) != 0;
    }
    if (!live) return;
    // the codes go by the scale as it is held
    float s = ZEROS ? __fdiv_rn(hi, 15.0f) - __fdiv_rn(lo, 15.0f) : __fdiv_rn(fmaxf(hi, -lo), 7.0f);
    if (!scales_f32) s = bf16w_lo(pack2_bf16(s, 0.0f));
    if (s == 0.0f) s = 1.0f;
    if (bad) s = __uint_as_float(0x7FC00000u);
    const float zero = ZEROS ? fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.0f), 15.0f) : 8.0f;
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float c = fminf(fmaxf(rintf(__fdiv_rn(x[k], s)) + zero, 0.0f), 15.0f);
        word |= static_cast<uint32_t>(c) << (4 * k);
    }
    codes[i] = word;
    if (i % lanes == 0) {
        const int64_t g = i / lanes;
        if (scales_f32) static_cast<float*>(scales)[g] = s;
        else static_cast<bf16_t*>(scales)[g] = static_cast<bf16_t>(__float_as_uint(s) >> 16);
        if constexpr (ZEROS) zeros[g] = static_cast<uint8_t>(zero);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int MT, int NT, int GROUP, X KIND, int WAVES>
hipError_t run(const LinearQ4Args& a, hipStream_t s) {
    const int64_t n_blocks = ceil_div(a.w.out, 16 * NT), m_blocks = ceil_div(a.rows, 16 * MT);
    const int64_t blocks = m_blocks > 1 ? ceil_div(n_blocks, 8) * 8 * m_blocks : n_blocks;
    if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
    const bool vec = aligned16(a.x) && a.x_stride % (KIND == X::kBf16 ? 8 : 4) == 0;
    hipLaunchKernelGGL((k_linear_q4<MT, NT, GROUP, KIND, WAVES>), dim3(static_cast<unsigned>(blocks)),
                       dim3(64 * WAVES), 0, s, a, vec, static_cast<int>(n_blocks), static_cast<int>(m_blocks));
    return hipGetLastError();
}

template <int GROUP>
hipError_t by_rows(const LinearQ4Args& a, bool f32, hipStream_t s) {
    if (f32 && a.rows <= kPackRows) return run<1, 1, GROUP, X::kPack, 8>(a, s);
    if (f32) {
        if (a.rows <= 16) return run<1, 2, GROUP, X::kTerms, 8>(a, s);
        if (a.rows <= 32) return run<2, 2, GROUP, X::kTerms, 8>(a, s);
        return run<4, 2, GROUP, X::kTerms, 8>(a, s);
    }
    if (a.rows <= 16) return run<1, 1, GROUP, X::kBf16, 8>(a, s);
    if (a.rows <= 32) return run<2, 2, GROUP, X::kBf16, 8>(a, s);
    return run<4, 2, GROUP, X::kBf16, 8>(a, s);
}

}  // namespace

size_t linear_q4_term_bytes(int64_t rows, int in, int, bool f32) {
    return f32 && rows > kPackRows ? static_cast<size_t>(rows) * in * 6 : 0;
}

hipError_t launch_linear_q4(const LinearQ4Args& a, bool f32, hipStream_t s) {
    if (a.rows <= 0 || a.w.out <= 0) return hipSuccess;
    if (a.terms) {
        const int64_t blocks = ceil_div(a.rows * (a.w.in / 8), 256);
        if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
        hipLaunchKernelGGL(k_q4_terms, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s,
                           static_cast<const float*>(a.x), a.x_stride, a.rows, a.w.in,
                           aligned16(a.x) && a.x_stride % 4 == 0, a.terms);
    }
    if (a.w.group == 32) return by_rows<32>(a, f32, s);
    if (a.w.group == 64) return by_rows<64>(a, f32, s);
    return by_rows<128>(a, f32, s);
}

hipError_t launch_quantise_q4(const void* w, bool w_f32, int64_t out, int in, int group, uint8_t* codes,
                              void* scales, bool scales_f32, uint8_t* zeros, hipStream_t s) {
    const int64_t runs = out * (in / 8), blocks = ceil_div(runs, 256);
    if (runs <= 0) return hipSuccess;
    if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(blocks)), block(256);
    uint32_t* to = reinterpret_cast<uint32_t*>(codes);
    const int lanes = group / 8;
    if (w_f32 && zeros) hipLaunchKernelGGL((k_quantise_q4<true, true>), grid, block, 0, s, w, runs, lanes, to, scales, scales_f32, zeros);
    else if (w_f32) hipLaunchKernelGGL((k_quantise_q4<true, false>), grid, block, 0, s, w, runs, lanes, to, scales, scales_f32, zeros);
    else if (zeros) hipLaunchKernelGGL((k_quantise_q4<false, true>), grid, block, 0, s, w, runs, lanes, to, scales, scales_f32, zeros);
    else hipLaunchKernelGGL((k_quantise_q4<false, false>), grid, block, 0, s, w, runs, lanes, to, scales, scales_f32, zeros);
    return hipGetLastError();
}

}  // namespace aps
