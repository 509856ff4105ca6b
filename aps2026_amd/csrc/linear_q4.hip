// Linear layers with weights in 4 bits (aps_linear_q4): y = x W^T + b with
// W[n][k] = (code - zero) scale, a scale and a zero for each `group` inputs; and
// aps_quantise_q4, which makes such weights.  Few rows here, many in
// linear_q4_many.hip.
//
// The matrix cores do the products for one row as for many: they take the codes
// with the fewest instructions.  A code c becomes the bf16 value 1 + c / 16 by
// putting its bits below an exponent (a shift and an and-or for two), and
//   sum_k x (c - zero) scale = 16 scale (sum_k x (1 + c / 16) - (1 + zero / 16) sum_k x)
// over each group.  All products are exact, sums are fp32.  An offset of 16 + zero
// codes, not the 128 of codes in the lowest bits, costs the fp32 sums 2 to 3 bits
// of a group's own sum: about 2e-7 of y where an fp32 chain over the inputs has
// 6e-7.
//
// fp32 x is the sum of three bf16 terms (8 bits each, cut off one after the
// other), so its products are exact too.  A group's sums are below
// 128 (1 + 255 / 16) of its largest x: finite up to 2^116.  Of x below 2^-110 the
// last bits are lost, those under bf16's smallest number, 2^-133.  Up to five rows
// have their terms below each other as rows of the matrix cores' 16.
//
// A lane loads 16 bytes, 32 codes of a row; the four lanes of a row hold 128
// neighbouring codes, so four swaps between the lanes' quarters (a 4 x 4
// transpose of words) give every product step 32 neighbouring inputs, the
// smallest group.  Within a lane's word of 8 codes the pairs of a register are
// (i, i + 4); x is put in the same order.
//
// Few rows of a wide weight are bound by the codes' bytes (one on 4096 x 32064 17.0
// us, 4.4 TB/s, of which some 4 are the start of the launch), of a narrow one by
// that start; what bounds more rows stands in linear_q4_many.hip.
#include <algorithm>

#include "q4.hpp"

namespace aps {
namespace {

using namespace q4;

constexpr int kPackRows = 5;     // fp32 rows whose three terms fit in 16
constexpr int kWaves = 16;       // one workgroup of 16 waves on a CU
constexpr int kFew = 64 * kWaves;
constexpr int kLds = 156 * 1024;

// LDS of a launch with 2^turns waves along the inputs: x, its sums, the waves'
// scales and zeros.
struct FewLds {
    int pitch;                   // bytes of a row of x
    int64_t x, sums, scales;     // bytes
};
__host__ __device__ inline FewLds few_lds(int rows, int in, int group, int turns, bool scales32) {
    const int pieces = (in + kPiece - 1) / kPiece, held = ((pieces + (1 << turns) - 1) >> turns) << turns;
    FewLds l;
    l.pitch = held * kPiece * 2 + kPad;
    l.x = static_cast<int64_t>(rows) * l.pitch;
    l.sums = static_cast<int64_t>(held) * (kPiece / group) * 64;
    l.scales = kWaves * 16 * (kBlock * (scales32 ? 4 : 2) + kPad + kBlock);
    return l;
}

// 2^columns waves lie side by side, 16 outputs each; the others share the inputs, a
// run of pieces each.  All of x lies in LDS.
//
// Rows of x in LDS: bf16 as they are, up to 16; fp32 a row's three terms below each
// other, up to five.  Row m of these is row 4 (m % 4) + m / 4 of the matrix cores'
// 16, so that up to four (NARROW) are register 0 of every lane and the others are
// not joined.
//
// A launch lasts little longer than its code takes to come from memory (10 KB
// more of it: 2 us), so loops stay loops.
template <int GROUP, bool F32, bool SCALES32, bool NARROW>
__global__ void __launch_bounds__(kFew) k_q4_few(LinearQ4Args a, int columns) {
    constexpr int GROUPS = kPiece / GROUP, STEPS = GROUP / 32;  // of a piece; product steps of a group
    constexpr int REGS = NARROW ? 1 : 4, BLOCK = kBlock / GROUPS;   // pieces of a block of scales
    constexpr int AHEAD = F32 ? 2 : 4;   // runs of x that a lane loads at once: 16 registers
    __shared__ __align__(16) unsigned char lds[kLds];
    const int tid = threadIdx.x, wave = tid / 64, lane = tid & 63, col = lane & 15, q = lane >> 4;
    const int wn = wave & ((1 << columns) - 1), wk = wave >> columns, log_turns = 4 - columns;
    const int in = a.w.in, pieces = (in + kPiece - 1) / kPiece, m_rows = static_cast<int>(a.rows);
    const int rounds = (pieces + (1 << log_turns) - 1) >> log_turns, rows = F32 ? 3 * m_rows : m_rows;
    const FewLds l = few_lds(rows, in, GROUP, log_turns, SCALES32);
    const int x_row = min(4 * (col & 3) + (col >> 2), rows - 1) * l.pitch + 16 * q;
    float* sums = reinterpret_cast<float*>(lds + l.x);   // [group][16]
    const CodeBits bits = code_bits();

    // Runs of 8 inputs go to lanes in units of 64 of a row.
    struct Run {
        float v[F32 ? 8 : 1];
        u32x4 w;
    };
    const int runs = (rounds << log_turns) * (kPiece / 8), units = (runs + 63) / 64;
    auto load_run = [&](int unit) {   // no branch
        Run r{};
        const int m = min(unit / units, m_rows - 1), run = unit % units * 64 + lane;
        const int64_t at = m * a.x_stride + begin_of(run / 32, run & 31, in).k;
        if constexpr (F32) load8(static_cast<const float*>(a.x) + at, r.v);
        else r.w = load8(static_cast<const bf16_t*>(a.x) + at);
        return r;
    };
    auto store_run = [&](int unit, Run r) {
        const int m = unit / units, run = unit % units * 64 + lane;
        if (m >= m_rows) return;   // the wave's all
        const Begin b = begin_of(run / 32, run & 31, in);
        if (b.k < b.at) r = Run{};
        float* to = sums + run / (GROUP / 8) * 16;
        auto place = [](int row) { return 4 * (row & 3) + (row >> 2); };
        if constexpr (F32) {
            u32x4 t[3];
            float sum[3];
            terms_of(r.v, t, sum);
#pragma unroll
            for (int e = 0; e < 3; ++e) sum[e] = add_lanes<GROUP / 8>(sum[e]);
            if (run >= runs) return;
#pragma unroll
            for (int e = 0; e < 3; ++e) {
                *reinterpret_cast<u32x4*>(lds + 16 * run + (3 * m + e) * l.pitch) = t[e];
                to[place(3 * m + e)] = sum[e];
            }
        } else {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += bf16w_lo(r.w[i]) + bf16w_hi(r.w[i]);
            sum = add_lanes<GROUP / 8>(sum);
            if (run >= runs) return;
            *reinterpret_cast<u32x4*>(lds + 16 * run + m * l.pitch) = code_order(r.w);
            to[place(m)] = sum;
        }
    };

    using Weight = Columns<1, GROUP, SCALES32>;
    const Weight w(a.w, ((static_cast<int>(blockIdx.x) << columns) + wn) * 16, lane, lds + l.x + l.sums + wave * Weight::LDS);
    const int first = wk * rounds, last = min(first + rounds, pieces);   // this wave's pieces
    float total[REGS] = {};
    // x before the codes, which come in order: it goes to LDS while they are on their way
    Run ahead[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) ahead[j] = load_run(wave + j * kWaves);
    Held<1> h0 = w.fetch(min(first, last - 1)), h1 = w.fetch(min(first + 1, last - 1));
    int block = w.load_scales(first);   // the first group of the scales in LDS
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) store_run(wave + j * kWaves, ahead[j]);
#pragma unroll 1
    for (int unit = wave + AHEAD * kWaves; unit < m_rows * units; unit += AHEAD * kWaves) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) ahead[j] = load_run(unit + j * kWaves);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) store_run(unit + j * kWaves, ahead[j]);
    }
    lds_barrier();
#pragma unroll 1
    for (int begin = first; begin < last; begin += BLOCK) {
        if (begin > first) block = w.load_scales(begin);
        const int end = min(begin + BLOCK, last);
#pragma unroll 1
        for (int piece = begin; piece < end; ++piece) {
            const Held<1> h = h0;
            h0 = h1;
            h1 = w.fetch(min(piece + 2, last - 1));
            const unsigned char* x = lds + x_row + piece * (kPiece * 2);
            const float* sum = sums + piece * GROUPS * 16 + 4 * q;
            const auto of = w.scales(w.first_group(piece) - block);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const u32x4 code = to_columns(h.code[c][0], lane);
#pragma unroll
                for (int g = c * (128 / GROUP); g < (c + 1) * (128 / GROUP); ++g) {
                    f32x4 dot = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int t = g * STEPS; t < (g + 1) * STEPS; ++t)
                        dot = mfma(frag(*reinterpret_cast<const u32x4*>(x + 64 * t)), code_values(code[t & 3], bits), dot);
#pragma unroll
                    for (int r = 0; r < REGS; ++r)
                        total[r] = fmaf(of.scale(0, g), fmaf(of.off(0, g), sum[16 * g + r], dot[r]), total[r]);
                }
            }
        }
    }
    // join the waves of the same columns in a fixed order
    lds_barrier();
    float* red = reinterpret_cast<float*>(lds);   // [wave][register][lane]
#pragma unroll
    for (int r = 0; r < REGS; ++r) red[(wave * REGS + r) * 64 + lane] = total[r];
    lds_barrier();
#pragma unroll 1
    for (int i = tid; i < m_rows << (columns + 4); i += kFew) {
        const int m = i >> (columns + 4), c = i & ((16 << columns) - 1);
        const int at = (static_cast<int>(blockIdx.x) << (columns + 4)) + c;
        if (at >= a.w.out) continue;
        // row m lies in register m / 4 of the lanes 16 (m % 4) ..
        auto of = [&](int wv, int row) { return red[(wv * REGS + (NARROW ? 0 : row >> 2)) * 64 + 16 * (row & 3) + (c & 15)]; };
        float y = 0.0f;
#pragma unroll 4
        for (int wv = c >> 4; wv < kWaves; wv += 1 << columns) {
            if constexpr (F32) {
#pragma unroll
                for (int t = 2; t >= 0; --t) y += of(wv, 3 * m + t);
            } else {
                y += of(wv, m);
            }
        }
        y *= 16.0f;
        if (a.bias) y += a.bias[at];
        const int64_t to = static_cast<int64_t>(m) * a.w.out + at;
        if constexpr (F32) static_cast<float*>(a.y)[to] = y;
        else static_cast<bf16_t*>(a.y)[to] = static_cast<bf16_t>(pack2_bf16(y, 0.0f) & 0xFFFFu);
    }
}

// Eight neighbouring values of a weight's row to a thread, its group's in
// neighbouring lanes.  32064 x 4096 takes 127 us from fp32 (4.7 TB/s) and 109 from
// bf16 (3.1 TB/s), whose bytes are little more than half: the divisions, one a
// value, count as much as they.
template <bool F32, bool ZEROS>
__global__ void __launch_bounds__(256)
k_quantise_q4(const void* __restrict__ w, int64_t runs, int lanes, uint32_t* __restrict__ codes, void* scales,
              bool scales_f32, uint8_t* zeros) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const bool live = i < runs;   // whole groups leave together, but the lanes' exchange needs all
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
        if constexpr (F32) {
            load8(static_cast<const float*>(w) + 8 * i, x);
        } else {
            const u32x4 v = load8(static_cast<const bf16_t*>(w) + 8 * i);
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

// The waves side by side: as many as leave every CU a workgroup (4096 x 32064, one
// row: 8 of them 15.7 us, 4 19.6, 16 23.7; 4096 x 6400: 2 7.3 us, 1 10.7, 4 9.1).
// -1, the other kernels, where x is too large for this one, and with bf16 rows past
// eight where x stays the longer part: a wave alone on its columns (16 rows on
// 2048 x 4096: 8.9 us here, 7.5 there; 12 on 4096 x 4096 9.0 either way; on
// 4096 x 8192 11.1 here, 12.1 there).  fp32 rows take 10 to 28 us there for 6 to 18.
int few_columns(const Q4& w, int64_t rows, bool f32) {
    if (rows > (f32 ? kPackRows : 16)) return -1;
    const int64_t tiles = ceil_div(w.out, 16);
    int columns = 0;
    while (columns < 4 && 256 << columns < tiles) ++columns;
    if (!f32 && rows > 8 && columns == 0) return -1;
    const FewLds l = few_lds(static_cast<int>(f32 ? 3 * rows : rows), w.in, w.group, 4 - columns, w.scales_f32);
    return l.x + l.sums + l.scales <= kLds ? columns : -1;
}

template <int GROUP, bool F32>
hipError_t run_few(const LinearQ4Args& a, int columns, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(ceil_div(a.w.out, 16 << columns))), block(kFew);
    const bool narrow = a.rows * (F32 ? 3 : 1) <= 4;
    if (narrow && a.w.scales_f32) hipLaunchKernelGGL((k_q4_few<GROUP, F32, true, true>), grid, block, 0, s, a, columns);
    else if (narrow) hipLaunchKernelGGL((k_q4_few<GROUP, F32, false, true>), grid, block, 0, s, a, columns);
    else if (a.w.scales_f32) hipLaunchKernelGGL((k_q4_few<GROUP, F32, true, false>), grid, block, 0, s, a, columns);
    else hipLaunchKernelGGL((k_q4_few<GROUP, F32, false, false>), grid, block, 0, s, a, columns);
    return hipGetLastError();
}

}  // namespace

size_t linear_q4_bytes(const Q4& w, int64_t rows, bool f32) {
    return rows <= 0 || few_columns(w, rows, f32) >= 0 ? 0 : q4_many_bytes(w, rows, f32);
}

hipError_t launch_linear_q4(const LinearQ4Args& a, bool f32, hipStream_t s) {
    if (a.rows <= 0 || a.w.out <= 0) return hipSuccess;
    const int columns = few_columns(a.w, a.rows, f32);
    if (columns < 0) return launch_q4_many(a, f32, s);
    if (a.w.group == 32) return f32 ? run_few<32, true>(a, columns, s) : run_few<32, false>(a, columns, s);
    if (a.w.group == 64) return f32 ? run_few<64, true>(a, columns, s) : run_few<64, false>(a, columns, s);
    return f32 ? run_few<128, true>(a, columns, s) : run_few<128, false>(a, columns, s);
}

template <bool F32, bool ZEROS>
static void quantise(const void* w, int64_t runs, int lanes, uint32_t* codes, void* scales, bool scales_f32,
                     uint8_t* zeros, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(ceil_div(runs, 256))), block(256);
    hipLaunchKernelGGL((k_quantise_q4<F32, ZEROS>), grid, block, 0, s, w, runs, lanes, codes, scales, scales_f32, zeros);
}

hipError_t launch_quantise_q4(const void* w, bool w_f32, int64_t out, int in, int group, uint8_t* codes,
                              void* scales, bool scales_f32, uint8_t* zeros, hipStream_t s) {
    const int lanes = group / 8;
    const int64_t runs = out * (in / 8), most = most_blocks(256) * 256;   // whole groups to a launch
    for (int64_t first = 0; first < runs; first += most) {
        const int64_t n = std::min(most, runs - first), groups = first / lanes;
        const void* from = static_cast<const char*>(w) + first * (w_f32 ? 32 : 16);
        uint32_t* to = reinterpret_cast<uint32_t*>(codes) + first;
        void* sc = static_cast<char*>(scales) + groups * (scales_f32 ? 4 : 2);
        if (w_f32 && zeros) quantise<true, true>(from, n, lanes, to, sc, scales_f32, zeros + groups, s);
        else if (w_f32) quantise<true, false>(from, n, lanes, to, sc, scales_f32, nullptr, s);
        else if (zeros) quantise<false, true>(from, n, lanes, to, sc, scales_f32, zeros + groups, s);
        else quantise<false, false>(from, n, lanes, to, sc, scales_f32, nullptr, s);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace aps
