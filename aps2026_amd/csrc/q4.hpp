// What the kernels of linear layers with 4-bit weights share: codes as operands of
// the matrix cores, and a wave's columns of a weight.
#pragma once

#include <type_traits>

#include "serve.hpp"

namespace aps {
namespace q4 {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kPiece = 256;   // inputs of a wave's turn: a 128-byte line of a row's codes
constexpr int kBlock = 16;    // groups whose scales and zeros a wave holds in LDS
constexpr int kPad = 16;      // bytes behind a row in LDS: other banks for the next

// Bytes at any address, in words; what is written as one number of them is read as
// another, so they may be aliases of anything.
template <int BYTES>
struct __attribute__((packed, aligned(1), may_alias)) Packed {
    uint32_t w[(BYTES + 3) / 4];
    __device__ uint32_t get4(int i) const { return w[i]; }
    __device__ uint32_t get2(int i) const { return (w[i / 2] >> (16 * (i & 1))) & 0xFFFFu; }
    __device__ uint32_t get1(int i) const { return (w[i / 4] >> (8 * (i & 3))) & 0xFFu; }
};
template <>
struct __attribute__((packed, aligned(1), may_alias)) Packed<2> {
    uint16_t w;
    __device__ uint32_t get1(int i) const { return (w >> (8 * i)) & 0xFFu; }
};

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

// Eight codes as bf16 1 + c / 16: (0, 4), (1, 5), (2, 6), (3, 7).  The constants are
// held in registers, where an and and an or of both are one instruction (as
// literals they would be two: 3 instructions a pair, not 2).
struct CodeBits {
    uint32_t mask, one;
};
__device__ inline CodeBits code_bits() {
    CodeBits b = {0x00780078u, 0x3F803F80u};
    asm("" : "+s"(b.mask));
    asm("" : "+v"(b.one));
    return b;
}
__device__ inline bf16x8 code_values(uint32_t w, CodeBits b) {
    return frag(u32x4{((w << 3) & b.mask) | b.one, ((w >> 1) & b.mask) | b.one, ((w >> 5) & b.mask) | b.one,
                      ((w >> 9) & b.mask) | b.one});
}

// Eight neighbouring bf16 values in the codes' order.
__device__ inline u32x4 code_order(u32x4 w) {
    return u32x4{__builtin_amdgcn_perm(w[2], w[0], 0x05040100u), __builtin_amdgcn_perm(w[2], w[0], 0x07060302u),
                 __builtin_amdgcn_perm(w[3], w[1], 0x05040100u), __builtin_amdgcn_perm(w[3], w[1], 0x07060302u)};
}

// The three bf16 terms of eight fp32 values, in the codes' order, and the sum of
// each term's.  The first term's values have 8 bits, so their sums, and those of
// their products with codes, are all but exact: kept apart from the others' they
// leave the result's own rounding (one sum for all: 3 times the error).
__device__ inline void terms_of(const float (&x)[8], u32x4 (&t)[3], float (&sum)[3]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            t[j][i] = __builtin_amdgcn_perm(__float_as_uint(v[i + 4]), __float_as_uint(v[i]), 0x07060302u);
        sum[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float cut = j < 2 ? __uint_as_float(__float_as_uint(v[i]) & 0xFFFF0000u) : v[i];
            sum[j] += cut;
            v[i] -= cut;
        }
    }
}

// Eight values at any alignment of their type.
__device__ inline void load8(const float* p, float (&x)[8]) {
    const auto t = *reinterpret_cast<const Packed<32>*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(t.w[i]);
}
__device__ inline u32x4 load8(const bf16_t* p) {
    const auto t = *reinterpret_cast<const Packed<16>*>(p);
    return u32x4{t.w[0], t.w[1], t.w[2], t.w[3]};
}

// A barrier for what is in LDS alone: loads on their way stay on their way.
__device__ inline void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Codes of a piece, as they were loaded.
template <int NT>
struct Held {
    u32x4 code[2][NT];
};

// The words that lane (column n, quarter q) of the products wants, from the load's
// lane 4 n + q, then 32 neighbouring inputs to a register.
__device__ inline u32x4 to_columns(u32x4 loaded, int lane) {
    const int from = 16 * (lane & 15) + 4 * (lane >> 4);   // bytes
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(from, static_cast<int>(loaded[i])));
    return transpose_quarters(w);
}

// A wave's 16 NT columns of a weight.
//
// Four neighbouring lanes read 64 neighbouring bytes of a row: a load takes a
// cycle for each line that such four touch, and a lane of its own row each, as the
// products want them, takes four times as many (this alone took one row on 4096 x
// 32064 from 24 us to 20).  The words go to their lanes through LDS's crossbar.  Scales
// and zeros come 16 groups at a time into LDS of the wave's own, for the same
// reason.
//
// The last piece, if it is not whole, covers the last 256 inputs (x is 0 there for
// those that the piece before has); with fewer than 256 in all, a row's last codes
// are read again in their place (x is 0 there too, and so are the scales).
template <int NT, int GROUP, bool SCALES32>
struct Columns {
    static constexpr int GROUPS = kPiece / GROUP, SIZE = SCALES32 ? 4 : 2, EACH = kBlock / 4;
    static constexpr int ROW = kBlock * SIZE + kPad + kBlock;   // bytes of a row's scales and zeros
    static constexpr int LDS = 16 * NT * ROW;                   // of a wave

    const Q4& w;
    int lane, at0, at1;
    const uint8_t* code_row[NT];
    int64_t scale_at[NT];
    unsigned char* lds;

    __device__ Columns(const Q4& w, int column, int lane, unsigned char* lds) : w(w), lane(lane), lds(lds) {
        at0 = min(16 * (lane & 3), w.in / 2 - 16);
        at1 = min(64 + 16 * (lane & 3), w.in / 2 - 16);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int64_t n = min(column + 16 * j + (lane >> 2), w.out - 1);
            code_row[j] = w.codes + n * (w.in / 2);
            scale_at[j] = n * (w.in / GROUP) + EACH * (lane & 3);
        }
    }
    __device__ int first_input(int piece) const { return max(min(piece * kPiece, w.in - kPiece), 0); }
    __device__ int first_group(int piece) const { return first_input(piece) / GROUP; }
    // no branch: the loads in flight stay countable
    __device__ Held<NT> fetch(int piece) const {
        const int k = first_input(piece) / 2;
        Held<NT> h;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            h.code[0][j] = *reinterpret_cast<const u32x4*>(code_row[j] + k + at0);
            h.code[1][j] = *reinterpret_cast<const u32x4*>(code_row[j] + k + at1);
        }
        return h;
    }
    // The scales and zeros from a piece's first group on, which it returns; four lanes
    // to a row.
    __device__ int load_scales(int piece) const {
        const int group = first_group(piece);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            // those that there are: of the weight, or of a short row
            const int64_t at = scale_at[j] + group, end = static_cast<int64_t>(w.out) * (w.in / GROUP);
            const int left = w.in < kPiece ? w.in / GROUP - EACH * (lane & 3) : static_cast<int>(min(end - at, static_cast<int64_t>(EACH)));
            const uint8_t* sp = static_cast<const uint8_t*>(w.scales) + at * SIZE;
            unsigned char* to = lds + (16 * j + (lane >> 2)) * ROW;
            unsigned char *scale_to = to + EACH * SIZE * (lane & 3), *zero_to = to + kBlock * SIZE + kPad + EACH * (lane & 3);
            if (left >= EACH) {
                *reinterpret_cast<Packed<EACH * SIZE>*>(scale_to) = *reinterpret_cast<const Packed<EACH * SIZE>*>(sp);
                if (w.zeros) *reinterpret_cast<Packed<EACH>*>(zero_to) = *reinterpret_cast<const Packed<EACH>*>(w.zeros + at);
            } else {
#pragma unroll 1
                for (int i = 0; i < EACH; ++i) {
                    // x is 0 past them, and 0 has to be what it is multiplied with too: 0 times
                    // an infinity or a NaN of the next rows, or of what LDS held, is not
                    *reinterpret_cast<Packed<SIZE>*>(scale_to + i * SIZE) = i < left ? *reinterpret_cast<const Packed<SIZE>*>(sp + i * SIZE) : Packed<SIZE>{};
                    if (w.zeros && i < left) zero_to[i] = w.zeros[at + i];
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
        return group;
    }
    // The scales and -(1 + zero / 16) of a piece's groups in the lane's column.
    struct Scales {
        Packed<GROUPS * SIZE> s[NT];
        Packed<GROUPS> z[NT];
        bool zeros;
        __device__ float scale(int j, int g) const {
            if constexpr (SCALES32) return __uint_as_float(s[j].get4(g));
            else return __uint_as_float(s[j].get2(g) << 16);
        }
        __device__ float off(int j, int g) const {
            return zeros ? fmaf(static_cast<float>(z[j].get1(g)), -0.0625f, -1.0f) : -1.5f;
        }
    };
    __device__ Scales scales(int group) const {   // `group` from the first in LDS
        Scales r;
        r.zeros = w.zeros != nullptr;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const unsigned char* row = lds + (16 * j + (lane & 15)) * ROW;
            r.s[j] = *reinterpret_cast<const Packed<GROUPS * SIZE>*>(row + group * SIZE);
            r.z[j] = *reinterpret_cast<const Packed<GROUPS>*>(row + kBlock * SIZE + kPad + group);
        }
        return r;
    }
};

// Where the eight inputs of run `run` (of 32) of a piece begin in a row of `in`:
// the piece's own inputs, or below `at` where x counts as 0.
struct Begin {
    int at, k;
};
__device__ inline Begin begin_of(int piece, int run, int in) {
    const int at = piece * kPiece, back = in < kPiece ? 0 : max(at + kPiece - in, 0);
    const int k = at + 8 * run - back;
    return {k < in ? at : 0x7FFFFFFF, min(k, in - 8)};
}

// Sum over the lanes of a group's eight-input runs (4, 8 or 16 neighbours) in the
// order of the lanes' numbers' bits.
template <int LANES>
__device__ inline float add_lanes(float v) {
    auto dpp = [](float x, auto ctrl) {
        return __uint_as_float(static_cast<uint32_t>(
            __builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(x)), decltype(ctrl)::value, 0xF, 0xF, true)));
    };
    v += dpp(v, std::integral_constant<int, 0xB1>{});                            // quads: 1 0 3 2
    v += dpp(v, std::integral_constant<int, 0x4E>{});                            // quads: 2 3 0 1
    if constexpr (LANES > 4) v += dpp(v, std::integral_constant<int, 0x141>{});  // halves of 16 mirrored
    if constexpr (LANES > 8) v += dpp(v, std::integral_constant<int, 0x140>{});  // 16 mirrored
    return v;
}

}  // namespace q4

// Many rows (linear_q4_many.hip).
size_t q4_many_bytes(const Q4& w, int64_t rows, bool f32);
hipError_t launch_q4_many(const LinearQ4Args& a, bool f32, hipStream_t s);

}  // namespace aps
