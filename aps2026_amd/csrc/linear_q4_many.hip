// Linear layers with weights in 4 bits for many rows (and for few whose inputs do
// not fit the kernel of linear_q4.hip): the same products, in two launches.
//
// The first puts x into the order in which the matrix cores take it, fp32 x as
// three bf16 terms (the workspace holds it):
//   [16 rows][piece of 256 inputs][term][8 steps of 32 inputs][64 lanes][16 bytes],
//   then the sums of x, [16 rows][group][row], of fp32 x those of the first term
//   and those of the other two
// so that an operand is one load of neighbouring bytes.  In the second a wave
// multiplies 16 MT rows by 16 NT columns over its share of the pieces, and a
// workgroup's eight waves are joined in LDS.  x comes from L2 without a stay in
// LDS: waves beside each other have other inputs, not the same ones.
//
// Bound by those reads of x, 64 bytes a cycle and CU (64 rows on 8192 x 8192: 1 MB
// for every 32 columns, 6.8 us), and by the codes' bytes (7.6); a workgroup's start
// and end take as long as one to two of its pieces, the first launch and the way to
// the second 5 us: 23.5 in all, 366 TFLOP/s.  Of a prompt's rows every 32 columns
// read x again, of fp32 x, whose terms are three times the bytes and products, every
// 16: 10240 rows on 4096 x 2048 take 291 us in bf16 (591 TFLOP/s) and 1438 in fp32
// (119, of the result's); a library's product with weights held in the same type
// 179 and 1155.
#include <algorithm>

#include "q4.hpp"

namespace aps {
namespace {

using namespace q4;

constexpr int kWaves = 8;
constexpr int64_t kCus = 256;
constexpr int kMany = 64 * kWaves;

constexpr int piece_bytes(int terms) { return 8 * terms * 1024; }
// Groups of a row with those of its last piece that lie past the inputs.
__host__ __device__ inline int all_groups(int in, int group) { return (in + kPiece - 1) / kPiece * (kPiece / group); }
__host__ __device__ inline int64_t sums_at(int64_t rows, int in, int terms) {
    return (rows + 15) / 16 * ((in + kPiece - 1) / kPiece) * piece_bytes(terms);
}

// A wave to a group of 16 rows: lane (row, quarter) takes runs of 8 inputs, 32 of
// them apart, all of them loaded before the first is used.
template <bool F32, int GROUP>
__global__ void __launch_bounds__(256) k_q4_arrange(LinearQ4Args a, int64_t first_wave, int64_t waves) {
    constexpr int TERMS = F32 ? 3 : 1, STEPS = GROUP / 32;
    const int64_t at = first_wave + static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64;
    if (at >= waves) return;
    const int lane = threadIdx.x & 63, q = lane >> 4, in = a.w.in, groups = all_groups(in, GROUP);
    const int64_t tile = at / groups;
    const int group = static_cast<int>(at - tile * groups), piece = group * GROUP / kPiece;
    const int first = group * STEPS & 7;   // step of the piece
    const int64_t row = min(tile * 16 + (lane & 15), a.rows - 1) * a.x_stride;
    uint8_t* to = reinterpret_cast<uint8_t*>(a.terms) + (tile * ((in + kPiece - 1) / kPiece) + piece) * piece_bytes(TERMS);
    float v[F32 ? STEPS : 1][8];
    u32x4 w[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int k = begin_of(piece, 4 * (first + i) + q, in).k;
        if constexpr (F32) load8(static_cast<const float*>(a.x) + row + k, v[i]);
        else w[i] = load8(static_cast<const bf16_t*>(a.x) + row + k);
    }
    float sum = 0.0f, low = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const Begin b = begin_of(piece, 4 * (first + i) + q, in);
        u32x4 t[3];
        if constexpr (F32) {
            float of[3];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = b.k < b.at ? 0.0f : v[i][e];
            terms_of(v[i], t, of);
            sum += of[0];
            low += of[1] + of[2];
        } else {
            if (b.k < b.at) w[i] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += bf16w_lo(w[i][e]) + bf16w_hi(w[i][e]);
            t[0] = code_order(w[i]);
        }
#pragma unroll
        for (int e = 0; e < TERMS; ++e) *reinterpret_cast<u32x4*>(to + (8 * e + first + i) * 1024 + 16 * lane) = t[e];
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    float* sums = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.terms) + sums_at(a.rows, in, TERMS));
    if (lane < 16) sums[at * 16 + lane] = sum;
    if constexpr (F32) {
        low += __shfl_xor(low, 16);
        low += __shfl_xor(low, 32);
        if (lane < 16) sums[(waves + at) * 16 + lane] = low;
    }
}

// 2^columns of a workgroup's waves lie side by side, 16 NT outputs each; the others
// share the inputs, a run of pieces each.
template <int GROUP, bool F32, int MT, int NT, bool SCALES32>
__global__ void __launch_bounds__(kMany) k_q4_many(LinearQ4Args a, int columns, int n_blocks, int first_m, int m_blocks) {
    constexpr int GROUPS = kPiece / GROUP, STEPS = GROUP / 32, TERMS = F32 ? 3 : 1, BLOCK = kBlock / GROUPS;
    using Weight = Columns<NT, GROUP, SCALES32>;
    // a wave's scales and zeros, and its rows' sums: [tile][group of the block][row]
    constexpr int KINDS = F32 ? 2 : 1, OWN = Weight::LDS + KINDS * MT * kBlock * 64;   // sums of the first term, of the others
    constexpr int RED = kWaves * NT * MT * 4 * 64 * 4, SCALE = kWaves * OWN;
    __shared__ __align__(16) unsigned char lds[RED > SCALE ? RED : SCALE];
    const int tid = threadIdx.x, wave = tid / 64, lane = tid & 63, q = lane >> 4;
    const int wn = wave & ((1 << columns) - 1), wk = wave >> columns, log_turns = 3 - columns;
    // blocks of the same columns on one XCD (workgroups go round the eight)
    int nb = blockIdx.x, mb = first_m;
    if (m_blocks > 1) {
        const int turn = blockIdx.x / 8;
        nb = (turn / m_blocks) * 8 + (blockIdx.x & 7);
        mb += turn % m_blocks;
        if (nb >= n_blocks) return;
    }
    const int in = a.w.in, pieces = (in + kPiece - 1) / kPiece, rounds = (pieces + (1 << log_turns) - 1) >> log_turns;
    const int64_t last_tile = (a.rows - 1) / 16;
    const uint8_t* x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
        x[i] = reinterpret_cast<const uint8_t*>(a.terms) +
               min(static_cast<int64_t>(mb) * MT + i, last_tile) * pieces * piece_bytes(TERMS);
    const Weight w(a.w, ((nb << columns) + wn) * 16 * NT, lane, lds + wave * OWN);
    float* own_sums = reinterpret_cast<float*>(lds + wave * OWN + Weight::LDS);
    const float* sums = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.terms) + sums_at(a.rows, in, TERMS));
    const int groups = all_groups(in, GROUP);
    const CodeBits bits = code_bits();
    const int first = wk * rounds, last = min(first + rounds, pieces);
    f32x4 total[NT][MT] = {};
    if (first < last) {
        Held<NT> h0 = w.fetch(first), h1 = w.fetch(min(first + 1, last - 1));
#pragma unroll 1
        for (int begin = first; begin < last; begin += BLOCK) {
            const int block = w.load_scales(begin), end = min(begin + BLOCK, last);
            // 16 groups of 16 rows, the last of them again past a row's end
            const int mine = min(begin * GROUPS + (lane >> 2), groups - 1) * 16 + 4 * (lane & 3);
#pragma unroll
            for (int i = 0; i < KINDS * MT; ++i) {
                const int64_t tile = min(static_cast<int64_t>(mb) * MT + i % MT, last_tile) + i / MT * (last_tile + 1);
                reinterpret_cast<f32x4*>(own_sums)[64 * i + lane] = *reinterpret_cast<const f32x4*>(sums + tile * groups * 16 + mine);
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int piece = begin; piece < end; ++piece) {
                const auto of = w.scales(w.first_group(piece) - block);
                const int64_t at = static_cast<int64_t>(piece) * piece_bytes(TERMS);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    u32x4 code[NT];
#pragma unroll
                    for (int j = 0; j < NT; ++j) code[j] = to_columns(h0.code[c][j], lane);
#pragma unroll
                    for (int g = c * (128 / GROUP); g < (c + 1) * (128 / GROUP); ++g) {
                        f32x4 dot[NT][MT][KINDS] = {}, sum[MT][KINDS];
#pragma unroll
                        for (int i = 0; i < MT * KINDS; ++i)
                            sum[i % MT][i / MT] = *reinterpret_cast<const f32x4*>(own_sums + (i * kBlock + (piece - begin) * GROUPS + g) * 16 + 4 * q);
#pragma unroll
                        for (int e = 0; e < TERMS; ++e)
#pragma unroll
                            for (int t = g * STEPS; t < (g + 1) * STEPS; ++t) {
                                bf16x8 xs[MT];
#pragma unroll
                                for (int i = 0; i < MT; ++i)
                                    xs[i] = frag(*reinterpret_cast<const u32x4*>(x[i] + at + (8 * e + t) * 1024 + 16 * lane));
#pragma unroll
                                for (int j = 0; j < NT; ++j) {
                                    const bf16x8 v = code_values(code[j][t & 3], bits);
#pragma unroll
                                    for (int i = 0; i < MT; ++i) dot[j][i][e > 0] = mfma(xs[i], v, dot[j][i][e > 0]);
                                }
                            }
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int i = 0; i < MT; ++i)
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    float v = fmaf(of.off(j, g), sum[i][0][r], dot[j][i][0][r]);
                                    if constexpr (F32) v += fmaf(of.off(j, g), sum[i][1][r], dot[j][i][1][r]);
                                    total[j][i][r] = fmaf(of.scale(j, g), v, total[j][i][r]);
                                }
                    }
                }
                // behind this piece's x: loads come in order
                h0 = h1;
                h1 = w.fetch(min(piece + 2, last - 1));
            }
        }
    }
    // join the waves of the same columns in a fixed order
    lds_barrier();
    float* red = reinterpret_cast<float*>(lds);   // [wave][tile][row][column]
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                red[((wave * NT + j) * 16 * MT + 16 * i + 4 * q + r) * 16 + (lane & 15)] = total[j][i][r];
    lds_barrier();
    const int64_t m0 = static_cast<int64_t>(mb) * 16 * MT, left = a.rows - m0;
    const int m_rows = left < 16 * MT ? static_cast<int>(left) : 16 * MT, cols = (16 * NT) << columns;
#pragma unroll 1
    for (int i = tid; i < m_rows * cols / 4; i += kMany) {
        const int m = i / (cols / 4), c = (i - m * (cols / 4)) * 4, n = nb * cols + c;
        f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int wv = c / (16 * NT); wv < kWaves; wv += 1 << columns)
            y += *reinterpret_cast<const f32x4*>(red + ((wv * NT + c / 16 % NT) * 16 * MT + m) * 16 + (c & 15));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (n + e >= a.w.out) break;
            float v = y[e] * 16.0f;
            if (a.bias) v += a.bias[n + e];
            const int64_t to = (m0 + m) * a.w.out + n + e;
            if constexpr (F32) static_cast<float*>(a.y)[to] = v;
            else static_cast<bf16_t*>(a.y)[to] = static_cast<bf16_t>(pack2_bf16(v, 0.0f) & 0xFFFFu);
        }
    }
}

// Up to 16 rows on a wide weight: 16 waves, kSide of them side by side with 16
// outputs each, which share x through LDS.  Two pieces of it (one for each of the
// two shares of the inputs) are copied there while the two before are multiplied.
// A wave that loaded x for itself would read 8 or 24 KB from L2 for every 2 KB of
// codes (16 fp32 rows on 4096 x 32064: 40 us, 27.7 here, of which 5 for putting x in
// order).  What bounds it is neither HBM (15 us) nor copies (without them 2 us less)
// but a round's own length, products after reads of LDS; two tiles of columns to a
// wave, which halve those reads, measure the same (31).
constexpr int kSide = 8, kWide = 1024, kWideOut = 16384;

template <int GROUP, bool F32, bool SCALES32>
__global__ void __launch_bounds__(kWide) k_q4_wide(LinearQ4Args a) {
    constexpr int GROUPS = kPiece / GROUP, STEPS = GROUP / 32, TERMS = F32 ? 3 : 1, BLOCK = kBlock / GROUPS;
    using Weight = Columns<1, GROUP, SCALES32>;
    constexpr int KINDS = F32 ? 2 : 1, OWN = Weight::LDS + KINDS * kBlock * 64, STAGE = 2 * piece_bytes(TERMS), COPIES = STAGE / 1024 / 16;
    // two arrays: a read of one need not wait for copies into the other
    __shared__ __align__(1024) unsigned char even[STAGE], odd[STAGE];
    __shared__ __align__(16) unsigned char owns[16 * OWN];
    const int tid = threadIdx.x, wave = tid / 64, lane = tid & 63, q = lane >> 4, wn = wave % kSide, wk = wave / kSide;
    const int in = a.w.in, pieces = (in + kPiece - 1) / kPiece, rounds = (pieces + 1) / 2, groups = all_groups(in, GROUP);
    const uint8_t* x = reinterpret_cast<const uint8_t*>(a.terms);
    const float* sums = reinterpret_cast<const float*>(x + sums_at(a.rows, in, TERMS));
    const Weight w(a.w, (static_cast<int>(blockIdx.x) * kSide + wn) * 16, lane, owns + wave * OWN);
    float* own_sums = reinterpret_cast<float*>(owns + wave * OWN + Weight::LDS);
    const CodeBits bits = code_bits();
    const int first = wk * rounds, last = min(first + rounds, pieces);
    // round `round`'s two pieces, 1 KB a copy (past the last piece the last again)
    auto copy = [&](int round, unsigned char* to) {
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const int at = (i * 16 + wave) * 1024, half = at / piece_bytes(TERMS);
            const int piece = min(half * rounds + min(round, rounds - 1), pieces - 1);
            const uint8_t* from = x + static_cast<int64_t>(piece) * piece_bytes(TERMS) + at % piece_bytes(TERMS) + 16 * lane;
            // Written out, for the compiler would let every read of LDS wait for it; it has
            // no result in registers, and the waits below count it.
            const uint32_t base = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(
                reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)(to + at))));
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base), "v"(from) : "memory", "m0");
        }
    };
    f32x4 total = {0.0f, 0.0f, 0.0f, 0.0f};
    copy(0, even);
    Held<1> h0 = w.fetch(min(first, last - 1)), h1 = w.fetch(min(first + 1, last - 1));
    int block = 0, begin = first;
    auto step = [&](int round, const unsigned char* here, unsigned char* next, Held<1>& h) {
        const int piece = first + round;
        // the copies of these two pieces, which were issued before the two loads of codes in flight
        // (vmcnt 2, lgkmcnt 0; a fence would wait for those too)
        __builtin_amdgcn_s_waitcnt(0x0070 | 2);
        asm volatile("s_barrier" ::: "memory");
        copy(round + 1, next);
        const u32x4 codes[2] = {to_columns(h.code[0][0], lane), to_columns(h.code[1][0], lane)};
        h = w.fetch(min(piece + 2, last - 1));
        if (piece >= last) return;
        const unsigned char* xs = here + wk * piece_bytes(TERMS) + 16 * lane;
        const auto of = w.scales(w.first_group(piece) - block);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            f32x4 dot[KINDS] = {};
#pragma unroll
            for (int e = 0; e < TERMS; ++e)
#pragma unroll
                for (int t = g * STEPS; t < (g + 1) * STEPS; ++t)
                    dot[e > 0] = mfma(frag(*reinterpret_cast<const u32x4*>(xs + (8 * e + t) * 1024)),
                                      code_values(codes[t / 4][t & 3], bits), dot[e > 0]);
            const float* sum = own_sums + ((piece - begin) * GROUPS + g) * 16 + 4 * q;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = fmaf(of.off(0, g), sum[r], dot[0][r]);
                if constexpr (F32) v += fmaf(of.off(0, g), sum[16 * kBlock + r], dot[1][r]);
                total[r] = fmaf(of.scale(0, g), v, total[r]);
            }
        }
    };
#pragma unroll 1
    for (int round = 0; round < rounds;) {
        begin = first + round;
        block = w.load_scales(begin);
        const int mine = min(begin * GROUPS + (lane >> 2), groups - 1) * 16 + 4 * (lane & 3);
#pragma unroll
        for (int i = 0; i < KINDS; ++i)
            reinterpret_cast<f32x4*>(own_sums)[64 * i + lane] = *reinterpret_cast<const f32x4*>(sums + i * groups * 16 + mine);
        __builtin_amdgcn_wave_barrier();
        const int end = min(round + BLOCK, rounds);   // BLOCK is even: the arrays stay in turn
#pragma unroll 1
        for (;;) {
            step(round, even, odd, h0);
            if (++round == end) break;
            step(round, odd, even, h1);
            if (++round == end) break;
        }
    }
    // the copies past the last round, then the two shares of a column joined
    __builtin_amdgcn_s_waitcnt(0x0F70);
    lds_barrier();
    float* red = reinterpret_cast<float*>(owns);   // [wave][row][column]
    static_assert(OWN >= 16 * 16 * 4, "a wave's own LDS holds its sums");
#pragma unroll
    for (int r = 0; r < 4; ++r) red[(wave * 16 + 4 * q + r) * 16 + (lane & 15)] = total[r];
    lds_barrier();
#pragma unroll 1
    for (int i = tid; i < static_cast<int>(a.rows) * kSide * 16; i += kWide) {
        const int m = i / (kSide * 16), c = i % (kSide * 16), n = static_cast<int>(blockIdx.x) * kSide * 16 + c;
        if (n >= a.w.out) continue;
        float y = (red[((c / 16) * 16 + m) * 16 + c % 16] + red[((c / 16 + kSide) * 16 + m) * 16 + c % 16]) * 16.0f;
        if (a.bias) y += a.bias[n];
        const int64_t to = static_cast<int64_t>(m) * a.w.out + n;
        if constexpr (F32) static_cast<float*>(a.y)[to] = y;
        else static_cast<bf16_t*>(a.y)[to] = static_cast<bf16_t>(pack2_bf16(y, 0.0f) & 0xFFFFu);
    }
}

template <int GROUP, bool F32>
hipError_t run_wide(const LinearQ4Args& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(ceil_div(a.w.out, 16 * kSide))), block(kWide);
    if (a.w.scales_f32) hipLaunchKernelGGL((k_q4_wide<GROUP, F32, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_q4_wide<GROUP, F32, false>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <int GROUP, bool F32, int MT, int NT>
hipError_t run(const LinearQ4Args& a, hipStream_t s) {
    const int64_t pieces = ceil_div(a.w.in, kPiece);
    // No wave without a piece; beyond that the columns whose rounds of workgroups take
    // the least, in pieces: those of a wave and what a workgroup's start and end take.
    // In us with 1, 2, 4, 8 waves side by side: 256 bf16 rows on 2048 x 4096 19.8, 15.9,
    // 21.5, 32.1; 64 on 8192 x 8192 26.4, 34.3, 57, 102; 64 on 4096 x 32064 54.8, 42.1,
    // 37.1, 60.6; 32 fp32 rows on 4096 x 12000 44.7, 40.5, 68.5, 122.
    int columns = 0;
    while (columns < 3 && (kWaves >> columns) > pieces) ++columns;
    int64_t least = INT64_MAX;
    for (int c = columns; c <= 3; ++c) {
        const int64_t blocks = ceil_div(a.w.out, (16 * NT) << c) * ceil_div(a.rows, 16 * MT);
        const int64_t cost = ceil_div(blocks, (MT > 1 ? 1 : 2) * kCus) * (ceil_div(pieces, kWaves >> c) + (F32 ? 1 : 2));
        if (cost < least) least = cost, columns = c;
    }
    const int64_t n_blocks = ceil_div(a.w.out, (16 * NT) << columns), m_blocks = ceil_div(a.rows, 16 * MT);
    const int64_t across = ceil_div(n_blocks, 8) * 8, most = most_blocks(kMany) / across;
    for (int64_t first = 0; first < m_blocks; first += most) {
        const int n = static_cast<int>(n_blocks), f = static_cast<int>(first), m = static_cast<int>(std::min(most, m_blocks - first));
        const dim3 grid(static_cast<unsigned>(m > 1 ? across * m : n_blocks)), block(kMany);
        if (a.w.scales_f32) hipLaunchKernelGGL((k_q4_many<GROUP, F32, MT, NT, true>), grid, block, 0, s, a, columns, n, f, m);
        else hipLaunchKernelGGL((k_q4_many<GROUP, F32, MT, NT, false>), grid, block, 0, s, a, columns, n, f, m);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Up to 16 rows: k_q4_wide past kWideOut outputs (16 fp32 rows on 4096 x 16384 27.0 us
// there, 24.3 here; on 4096 x 20000 27.5 and 34.4; bf16 on 8192 x 16384 30.4 and 25.6,
// on 8192 x 24000 33.3 and 41.5).  More rows: 16 rows by 16 columns a wave with fp32 x,
// whose loads and products are thrice as many; with bf16 two or four times the rows and
// twice the columns where enough workgroups are left for the CUs.  In us with 64, 32 and
// 16 rows a tile, bf16:
//   64 rows on 4096 x 32064   37.1  41.1  61.7     64 rows on 4096 x 4096   15.1  12.7  14.2
//   256 on 2048 x 4096        15.4  15.6  18.4     64 rows on 8192 x 8192   25.1  24.0  30.7
//   256 on 2048 x 2048        12.2  11.4  12.8     32 rows on 4096 x 1024   13.3  10.4   7.9
// fp32 with 32 and 16:
//   64 rows on 4096 x 4096           25.8  23.6     17 rows on 4096 x 4096        24.3  17.1
//   256 on 2048 x 4096               42.9  37.3     32 rows on 4096 x 32064       73.8  67.1
template <int GROUP, bool F32>
hipError_t by_rows(const LinearQ4Args& a, hipStream_t s) {
    if (a.rows <= 16 && a.w.out > kWideOut) return run_wide<GROUP, F32>(a, s);
    if constexpr (!F32) {
        const auto workgroups = [&](int mt) { return ceil_div(a.rows, 16 * mt) * ceil_div(a.w.out, 32); };
        if (a.rows > 32 && workgroups(4) >= 2 * kCus) return run<GROUP, F32, 4, 2>(a, s);
        if (a.rows > 16 && workgroups(2) >= kCus) return run<GROUP, F32, 2, 2>(a, s);
    }
    return run<GROUP, F32, 1, 1>(a, s);
}

}  // namespace

size_t q4_many_bytes(const Q4& w, int64_t rows, bool f32) {
    return static_cast<size_t>(sums_at(rows, w.in, f32 ? 3 : 1) + ceil_div(rows, 16) * all_groups(w.in, w.group) * (f32 ? 128 : 64));
}

template <int GROUP>
static hipError_t launch(const LinearQ4Args& a, bool f32, hipStream_t s) {
    const int64_t waves = ceil_div(a.rows, 16) * all_groups(a.w.in, GROUP), most = most_blocks(256) * 4;
    for (int64_t first = 0; first < waves; first += most) {
        const dim3 grid(static_cast<unsigned>(ceil_div(std::min(most, waves - first), 4)));
        if (f32) hipLaunchKernelGGL((k_q4_arrange<true, GROUP>), grid, dim3(256), 0, s, a, first, waves);
        else hipLaunchKernelGGL((k_q4_arrange<false, GROUP>), grid, dim3(256), 0, s, a, first, waves);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return f32 ? by_rows<GROUP, true>(a, s) : by_rows<GROUP, false>(a, s);
}

hipError_t launch_q4_many(const LinearQ4Args& a, bool f32, hipStream_t s) {
    if (a.w.group == 32) return launch<32>(a, f32, s);
    return a.w.group == 64 ? launch<64>(a, f32, s) : launch<128>(a, f32, s);
}

}  // namespace aps
