// Attention of each sequence's newest tokens over its paged cache
// (aps_attention_paged): a sliding window plus the first tokens, fp32, bf16
// and 4-bit caches, any number of new tokens.
//
// The rows of a sequence under one key head are its (token, query head)
// pairs, token-major; a tile is 16 of them, and a wave walks 32 (fp32 cache:
// 16) keys a step with the products transposed:
//   S^T = K Q^T    16 keys x 16 rows, A = K, B = Q^T
//   O^T += V^T P^T  16 dims x 16 rows, A = V^T, B = P^T
// In the MFMA's result a lane holds one row (lane % 16) and, of group g =
// lane / 16, the keys 4 g + i; as B operand of the second product it has to
// hold 8 (fp32: 1) keys of that row, any ones as long as A holds the same: so
// the weights never leave their lane, the row's maximum and sum take two
// exchanges, and scaling the accumulator is one factor a lane.  K is read in
// MFMA layout; of V a lane reads head_dim / 16 neighbouring dims of 4 g + i's
// rows and turns them in registers (v_perm), column c of dim tile t being dim
// (head_dim / 16) c + t.  Nothing is staged in LDS: a key or value goes from
// HBM to the registers that multiply it, once per tile of rows.
//
// Numbers: the running maximum and sum are fp32 in base 2 (scores times scale
// log2 e).  fp32 queries against bf16 or 4-bit keys are split into three bf16
// terms (24 bits: exact products on the bf16 MFMAs), fp32 weights likewise;
// bf16 queries keep their weights to two terms (16 bits).  An fp32 cache runs
// on the fp32 MFMAs.
//
// A value that a row does not see must not reach it.  Scores of such keys are
// replaced; in the second product their weight is 0, but 0 times an infinity
// or a NaN is a NaN: rows of V that no row of the tile sees are replaced by
// zeros, and where rows differ in what they see, a row that ended in NaN is
// computed again from its own keys alone (redo_row) if a value that it does not
// see may be why (stray).
//
// Few rows and a long cache: the steps of a tile are split over the 4 to 8 waves
// of a workgroup and, past that, over `splits` workgroups; the waves' (max, sum,
// O) meet in LDS, the workgroups' in the workspace, joined by k_paged_join.
#include <algorithm>
#include <type_traits>

#include "serve.hpp"

namespace aps {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kMostWaves = 8;  // 256 registers a wave
constexpr int kRows = 16;      // rows of a tile
constexpr int kMaxSplits = 256, kFewSplits = 8;
constexpr int kPlainLds = 62 * 1024;  // dynamic LDS that needs no leave: 64 KB less the static part
// Rows of a sequence under a key head from which k_paged_tiles takes them.  us in
// k_paged_rows / k_paged_tiles, of 64 sequences on 1024 keys and of 2 on 8192:
//   36 rows  bf16 67 / 34, 26 / 18   fp32 on bf16 69 / 50, 29 / 25
//            4 bits 31 / 30, 16 / 17  fp32 cache 122 / 141, 47 / 48
//   20 rows  bf16 47 / 31, 15 / 17   fp32 on bf16 49 / 38, 17 / 24
//            4 bits 23 / 25, 12 / 16  fp32 cache 85 / 84, 25 / 46
// Below it k_paged_rows is ahead where there are few sequences or few bits, and
// holds weights to more of them.
constexpr int64_t kTiledRows = 33;

// What both kernels know of the launch.
struct PagedDev {
    PagedArgs a;
    KvCache c;
    int group;       // query heads per key head
    int page_shift;
    int splits;      // workgroups along the keys
    int row_tiles;   // tiles (tiled: blocks) of rows a sequence and key head can have
    bool tiled;      // k_paged_tiles, else k_paged_rows
    int least, most;  // rows of the sequences that this launch serves
    int64_t max_q;    // the most tokens of one
    bool by_seq;      // parts stand by (sequence, token), max_q of each, else by row of q
    int64_t slots;    // (sequence, token)s or rows that have parts
    int waves;       // of a workgroup
    int lds_rows;    // rows of a tile that can be live: LDS keeps those
    int64_t blocks;  // workgroups
    float* part;     // of the splits
    float scale_log2;
};
// The rows under one key head that a sequence has in this launch, 0 if it is
// another's.
__device__ inline int rows_of(const PagedDev& d, int len) {
    const int64_t n = (len < d.a.max_q_len ? len : d.a.max_q_len) * d.group;
    return n >= d.least && n <= d.most ? static_cast<int>(n) : 0;
}

// Rows q0 .. q0 + len - 1 and the cached length of a sequence, inside the arrays
// whatever the device values are.
struct Seq {
    int64_t q0;
    int len, kv;
};
__device__ inline Seq clipped(const PagedDev& d, int64_t lo, int64_t hi, int64_t kv) {
    Seq s;
    s.q0 = lo < 0 ? 0 : lo > d.a.rows ? d.a.rows : lo;
    const int64_t n = (hi < d.a.rows ? hi : d.a.rows) - s.q0;
    s.len = static_cast<int>(n < 0 ? 0 : n);
    const int64_t held = d.a.table_stride << d.page_shift;
    kv = kv < d.a.max_kv_len ? kv : d.a.max_kv_len;
    kv = kv < held ? kv : held;
    s.kv = static_cast<int>(kv < 0 ? 0 : kv);
    return s;
}
// Sequence b, the same in every lane (in scalar registers, and with it the
// places that loads start from).
__device__ inline Seq sequence(const PagedDev& d, int64_t b) {
    return clipped(d, __builtin_amdgcn_readfirstlane(d.a.q_offsets[b]),
                   __builtin_amdgcn_readfirstlane(d.a.q_offsets[b + 1]),
                   __builtin_amdgcn_readfirstlane(d.a.kv_lens[b]));
}

// The keys that the rows at positions [pmin, pmax] see, in steps of STEP keys:
// the first tokens' steps, then the window's.
struct Keys {
    int lo, hi, first;  // a key is seen by some row only if key < hi and (key >= lo or key < first)
    int n1, t_lo, steps;
};
template <int STEP>
__device__ inline Keys visible(const PagedDev& d, int pmin, int pmax) {
    Keys k;
    // (the division behind a position leaves scalar registers)
    pmin = __builtin_amdgcn_readfirstlane(pmin);
    pmax = __builtin_amdgcn_readfirstlane(pmax);
    k.hi = pmax + 1 > 0 ? pmax + 1 : 0;
    const int64_t lo = static_cast<int64_t>(pmin) + 1 - d.a.window;
    k.lo = lo > 0 ? static_cast<int>(lo) : 0;
    k.first = d.a.sinks < k.hi ? d.a.sinks : k.hi;
    k.t_lo = k.lo / STEP;
    const int t_hi = (k.hi + STEP - 1) / STEP;
    k.n1 = (k.first + STEP - 1) / STEP;
    if (k.n1 > k.t_lo) k.n1 = k.t_lo;
    k.steps = k.n1 + (t_hi > k.t_lo ? t_hi - k.t_lo : 0);
    return k;
}

// The page of the 16 keys 16 a .. of step t, -1 where there is none: behind the
// last key that is seen, past t1, or an id outside the cache.  A wave reads the
// pages of many steps at once, a lane each.
template <int STEP>
__device__ inline int page_of(const PagedDev& d, const int32_t* table, const Keys& ks, int t, int t1, int a) {
    const int key = (t < ks.n1 ? t : t - ks.n1 + ks.t_lo) * STEP + 16 * a;
    const int page = t < t1 && key < ks.hi ? table[key >> d.page_shift] : -1;
    return page >= 0 && page < d.c.num_pages ? page : -1;
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// A row's view of the keys: key <= pos and (key > low or key < sinks).
struct View {
    int pos, low;
};
__device__ inline View view(const PagedDev& d, int pos) {
    const int64_t low = static_cast<int64_t>(pos) - d.a.window;
    return View{pos, low > -1 ? static_cast<int>(low) : -1};
}
__device__ inline bool sees(const PagedDev& d, const View& v, int key) {
    return (key <= v.pos) & ((key > v.low) | (key < d.a.sinks));
}
// Maximum and sum over the lanes l, l ^ 16 and l, l ^ 32.
__device__ inline float max_x32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float max_x16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// x and the lanes c ^ 7 (row_half_mirror) or c ^ 8 (row_ror:8) of the 16: sums of
// the same two numbers in either lane.
template <int CTRL>
__device__ inline float plus_dpp(float x) {
    return x + __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xF, 0xF, true));
}
constexpr int kHalfMirror = 0x141, kRor8 = 0x128;
__device__ inline float less_bits(float x, uint32_t mask) { return x - __uint_as_float(__float_as_uint(x) & mask); }
__device__ inline float bf16_round(float x) { return __uint_as_float(pack2_bf16(x, 0.0f) << 16); }

// One cached element as fp32 (redo_row).
template <int D, Kv KV>
__device__ inline float element(const void* base, const uint8_t* scales, int64_t head_row, int dim) {
    if constexpr (KV == Kv::kF32) return static_cast<const float*>(base)[head_row * D + dim];
    if constexpr (KV == Kv::kBf16)
        return __uint_as_float(static_cast<uint32_t>(static_cast<const bf16_t*>(base)[head_row * D + dim]) << 16);
    const uint32_t byte = static_cast<const uint8_t*>(base)[head_row * (D / 2) + dim / 2];
    const uint32_t pair = mx_decode2<0>(byte, mx_scale(scales[head_row * (D / 32) + dim / 32]));
    return dim & 1 ? bf16w_hi(pair) : bf16w_lo(pair);
}

// True if a value that is not finite may have reached a row that does not see it:
// one of a key that other rows see, in a step of [t0, t1) that rows at positions
// [pmin, pmax] do not all see whole.  (Where they do, it is the row's own.)
template <int D, Kv KV, int STEP>
__device__ bool stray(const PagedDev& d, const int32_t* table, int h, const Keys& ks, int t0, int t1, int pmin,
                      int pmax, int pos) {
    const View vis = view(d, pos);
    const int lane = threadIdx.x & 63;
    bool found = false;
    for (int t = t0; t < t1 && !found; ++t) {
        const int base = (t < ks.n1 ? t : t - ks.n1 + ks.t_lo) * STEP;
        if (base + STEP - 1 <= pmin && (static_cast<int64_t>(base) > static_cast<int64_t>(pmax) - d.a.window ||
                                        base + STEP - 1 < d.a.sinks))
            continue;
        bool bad = false;
        for (int key = base; key < base + STEP && key < ks.hi; ++key) {
            if ((key < ks.lo && key >= ks.first) || sees(d, vis, key)) continue;
            const int64_t page = table[key >> d.page_shift];
            if (page < 0 || page >= d.c.num_pages) continue;
            const int64_t hr = ((page * d.c.kv_heads + h) << d.page_shift) + (key & ((1 << d.page_shift) - 1));
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                const float x = element<D, KV>(d.c.v, d.c.v_scale, hr, D / 64 * lane + j);
                bad |= x - x != 0.0f;
            }
        }
        found = __any(bad);
    }
    return found;
}

// One row over the steps [t0, t1) from the keys it sees alone, by a whole wave:
// 64 keys at a time, a lane the score of each, then the values one key after the
// other; o[dim], m and l in LDS.
template <int D, bool Q32, Kv KV, int STEP>
__device__ void redo_row(const PagedDev& d, const int32_t* table, int h, const Keys& ks, int t0, int t1, int64_t qrow,
                         int head, int pos, float* o, float* m_out, float* l_out) {
    constexpr int PER = D / 64;
    const View vis = view(d, pos);
    const int lane = threadIdx.x & 63;
    float q[PER], acc[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int64_t at = qrow * d.a.q_stride + static_cast<int64_t>(head) * D + PER * lane + j;
        q[j] = Q32 ? static_cast<const float*>(d.a.q)[at]
                   : __uint_as_float(static_cast<uint32_t>(static_cast<const bf16_t*>(d.a.q)[at]) << 16);
        acc[j] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int t = t0; t < t1; t += 64 / STEP) {
        const int mine = t + lane / STEP;
        const int key = (mine < ks.n1 ? mine : mine - ks.n1 + ks.t_lo) * STEP + lane % STEP;
        const bool seen = mine < t1 && sees(d, vis, key);
        const int64_t page = seen ? table[key >> d.page_shift] : -1;
        const bool held = page >= 0 && page < d.c.num_pages;
        const int64_t hr =
            held ? ((page * d.c.kv_heads + h) << d.page_shift) + (key & ((1 << d.page_shift) - 1)) : 0;
        float s = 0.0f;
        for (int x = 0; x < 64; ++x)
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const float qx = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(q[j]), x));
                s = fmaf(qx, held ? element<D, KV>(d.c.k, d.c.k_scale, hr, PER * x + j) : 0.0f, s);
            }
        s = held ? s * d.scale_log2 : -INFINITY;
        float top = s;
#pragma unroll
        for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.0f : mn;
        const float f = exp2_fast(m - ref), p = exp2_fast(s - ref);
        m = mn;
        float sum = p;
#pragma unroll
        for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x);
        l = l * f + sum;
#pragma unroll
        for (int j = 0; j < PER; ++j) acc[j] *= f;
        for (uint64_t left = __ballot(held); left; left &= left - 1) {
            const int x = __builtin_ctzll(left);
            const float px = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), x));
            const int64_t hx =
                static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(
                                         __builtin_amdgcn_readlane(static_cast<int>(hr >> 32), x)))
                                     << 32) |
                static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(hr), x));
#pragma unroll
            for (int j = 0; j < PER; ++j)
                acc[j] = fmaf(px, element<D, KV>(d.c.v, d.c.v_scale, hx, PER * lane + j), acc[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) o[PER * lane + j] = acc[j];
    if (lane == 0) { *m_out = m; *l_out = l; }
}

// SIDE: few rows (side_rows), whose terms stand side by side in the 16 columns of
// the MFMAs instead of one product after the other: column c holds term c / 4 of
// row c % 4 (mirrored where c & 4, for the sums over lanes c ^ 7), with BF16
// queries term c / 8 of row c % 8.  Scores are summed over a row's columns, which
// then hold the same weight and take their term of it; O is summed at the end.
// (One sequence of 131072 4-bit keys, fp32 queries: 27.0 -> 24.7 us; 64 of 16384:
// 113 -> 94, with BF16 queries 91 -> 89; a bf16 cache is bound by its bytes.)
// The rows that 16 columns hold beside each other: of four terms, of two.
constexpr int side_rows(bool q32) { return q32 ? 4 : 8; }

template <int D, bool Q32, Kv KV, bool SIDE>
__global__ void __launch_bounds__(64 * kMostWaves, 2)
k_paged_rows(PagedDev d) {
    constexpr bool FP = KV == Kv::kF32;
    constexpr int HALVES = FP ? 1 : 2;
    constexpr int STEP = 16 * HALVES;
    constexpr int W = D / 16;          // dims of V a lane reads of a key, and dim tiles
    constexpr int QT = Q32 && !SIDE ? 3 : 1;        // products a query's bf16 terms take
    constexpr int PT = SIDE ? 1 : Q32 ? 3 : 2;      // and a weight's
    constexpr int KS = D / 32;         // MFMA steps over the dims
    constexpr int OSTRIDE = D + 4;     // LDS row, off the banks' period
    __shared__ float sm_m[kMostWaves][kRows], sm_l[kMostWaves][kRows];
    extern __shared__ __align__(16) float sm_o[];  // [waves][lds_rows][OSTRIDE]
    auto o_row = [&](int w, int r) { return sm_o + (w * d.lds_rows + r) * OSTRIDE; };

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    uint32_t id = blockIdx.x;
    const int split = __builtin_amdgcn_readfirstlane(id % d.splits);
    id /= d.splits;
    const int rt = __builtin_amdgcn_readfirstlane(id % d.row_tiles);
    id /= d.row_tiles;
    const int h = __builtin_amdgcn_readfirstlane(id % d.c.kv_heads);
    const int64_t b = __builtin_amdgcn_readfirstlane(id / d.c.kv_heads);
    const Seq sq = sequence(d, b);
    const int nrows = rows_of(d, sq.len);
    const int r0 = rt * kRows;
    if (r0 >= nrows) return;  // the whole workgroup
    const int32_t* table = d.a.page_table + b * d.a.table_stride;

    const int p0 = sq.kv - sq.len;  // position of the first new token
    const int r_last = r0 + kRows - 1 < nrows ? r0 + kRows - 1 : nrows - 1;
    const int pmin = __builtin_amdgcn_readfirstlane(p0 + r0 / d.group);
    const int pmax = __builtin_amdgcn_readfirstlane(p0 + r_last / d.group);
    const int term = !SIDE ? 0 : Q32 ? c >> 2 : c >> 3;
    const int row = r0 + (!SIDE ? c : !Q32 ? c & 7 : c & 4 ? 3 - (c & 3) : c & 3);
    const bool live = row < nrows;
    const int tok = live ? row / d.group : 0, qh = h * d.group + (live ? row % d.group : 0);
    const int pos = live ? p0 + tok : -1;
    // what of a weight a term leaves out: 8 leading bits a term before it
    const uint32_t out1 = term == 0 ? 0u : term == 3 ? ~0u : 0xFFFF0000u, out2 = term == 2 ? 0xFFFF0000u : 0u;
    const Keys ks = visible<STEP>(d, pmin, pmax);
    const int parts = d.splits * d.waves, part = split * d.waves + wave;
    const int each = __builtin_amdgcn_readfirstlane((ks.steps + parts - 1) / parts);
    const int t0 = part * each < ks.steps ? part * each : ks.steps;
    const int t1 = t0 + each < ks.steps ? t0 + each : ks.steps;

    // the queries, in the order of dims that the cache's loads give
    f32x4 qf[FP ? D / 16 : 1];
    bf16x8 qb[FP ? 1 : QT][FP ? 1 : KS];
    {
        const int64_t qat = (sq.q0 + tok) * d.a.q_stride + static_cast<int64_t>(qh) * D;
        if constexpr (FP) {
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
                qf[s] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(d.a.q) + qat + 16 * s + 4 * g);
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int dim = KV == Kv::kMx ? (D / 4) * g + 8 * s : 32 * s + 8 * g;
                if constexpr (Q32) {
                    const float* p = static_cast<const float*>(d.a.q) + qat + dim;
                    const f32x4 x0 = *reinterpret_cast<const f32x4*>(p), x1 = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float x = j < 4 ? x0[j & 3] : x1[j & 3];
                        if constexpr (SIDE) {
                            const float t0 = bf16_round(x), t1 = bf16_round(x - t0), t2 = bf16_round(x - t0 - t1);
                            qb[0][s][j] = static_cast<__bf16>(term == 0 ? t0 : term == 1 ? t1 : term == 2 ? t2 : 0.0f);
                            continue;
                        }
#pragma unroll
                        for (int t = 0; t < QT; ++t) {
                            const float hi = bf16_round(x);
                            qb[t][s][j] = static_cast<__bf16>(hi);
                            x -= hi;
                        }
                    }
                } else {
                    qb[0][s] = *reinterpret_cast<const bf16x8*>(static_cast<const bf16_t*>(d.a.q) + qat + dim);
                }
            }
        }
    }

    f32x4 acc[W];
#pragma unroll
    for (int t = 0; t < W; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;

    const View vis = view(d, pos);
    constexpr int AHEAD = 64 / HALVES;  // steps whose pages the lanes hold
    int pages = -1;
    // what a lane reads of a step: its part of K, of V, and 4-bit scale bytes
    constexpr bool MX = KV == Kv::kMx;
    constexpr int KW = FP ? D / 4 : MX ? 2 * KS : 8 * KS;   // words
    constexpr int VW = FP ? 4 * W : MX ? 8 : 4 * W;
    struct Step {
        bool dead[HALVES];  // no page
        uint32_t k[KW], v[VW], ks[MX ? 2 : 1], vs[MX ? 8 : 1];
    };
    auto words = [](const void* p, auto n, uint32_t* to) {
        constexpr int N = decltype(n)::value;
        if constexpr (N == 4) {
            const u32x4 w = *static_cast<const u32x4*>(p);
#pragma unroll
            for (int x = 0; x < 4; ++x) to[x] = w[x];
        } else {
            const u32x2 w = *static_cast<const u32x2*>(p);
            to[0] = w[0];
            to[1] = w[1];
        }
    };
    using Four = std::integral_constant<int, 4>;
    // a lane's bytes past the (uniform) place of 16 keys: a 32-bit offset and a
    // constant for each load
    const uint32_t k_lane = FP ? c * (4 * D) + 16 * g : MX ? c * (D / 2) + (D / 8) * g : c * (2 * D) + 16 * g;
    const uint32_t v_lane = FP ? 4 * g * (4 * D) + 4 * W * c : MX ? 4 * g * (D / 2) + (W / 2) * c
                                                                  : 4 * g * (2 * D) + 2 * W * c;
    const uint32_t ks_lane = c * (D / 32) + (D / 4) * g / 32, vs_lane = 4 * g * (D / 32) + W * c / 32;
    auto load = [&](int t, Step& st) {
        const int base = (t < ks.n1 ? t : t - ks.n1 + ks.t_lo) * STEP;
        const int slot = (t - t0) % AHEAD;
        if (slot == 0) pages = page_of<STEP>(d, table, ks, t + lane / HALVES, t1, lane % HALVES);
#pragma unroll
        for (int a = 0; a < HALVES; ++a) {
            const int page = __builtin_amdgcn_readlane(pages, slot * HALVES + a);
            st.dead[a] = page < 0;
            // (page, head, offset) row of the half's first key
            const int64_t hrow = ((static_cast<int64_t>(page < 0 ? 0 : page) * d.c.kv_heads + h) << d.page_shift) +
                                 ((base + 16 * a) & ((1 << d.page_shift) - 1));
            constexpr int BYTES = FP ? 4 * D : MX ? D / 2 : 2 * D;  // of a key
            const uint8_t* kp = static_cast<const uint8_t*>(d.c.k) + hrow * BYTES;
            const uint8_t* vp = static_cast<const uint8_t*>(d.c.v) + hrow * BYTES;
            if constexpr (FP) {
#pragma unroll
                for (int s = 0; s < D / 16; ++s) words(kp + k_lane + 64 * s, Four(), st.k + 4 * s);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < W; x += 4) words(vp + v_lane + BYTES * i + 4 * x, Four(), st.v + W * i + x);
            } else if constexpr (!MX) {
#pragma unroll
                for (int s = 0; s < KS; ++s) words(kp + k_lane + 64 * s, Four(), st.k + 4 * (KS * a + s));
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    words(vp + v_lane + BYTES * i, std::integral_constant<int, W / 2>(), st.v + (W / 2) * (4 * a + i));
            } else {
                // D / 4 neighbouring dims of a key of K: one block's, or half a block's
                words(kp + k_lane, std::integral_constant<int, KS>(), st.k + KS * a);
                st.ks[a] = (d.c.k_scale + hrow * (D / 32))[ks_lane];
                const uint8_t* sp = d.c.v_scale + hrow * (D / 32);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (W == 8) st.v[4 * a + i] = *reinterpret_cast<const uint32_t*>(vp + v_lane + BYTES * i);
                    else st.v[4 * a + i] = *reinterpret_cast<const uint16_t*>(vp + v_lane + BYTES * i);
                    st.vs[4 * a + i] = (sp + vs_lane)[i * (D / 32)];
                }
            }
        }
    };

    // A step is read one ahead (37 x 2051 fp32 keys 80 -> 63 us, 64 x 8192 bf16 154
    // -> 148; 64 x 16384 4-bit keys under fp32 rows 132 -> 111), except of a
    // 4-bit cache in the leaner variants, whose decoding wants the registers for a
    // third or fourth wave (the same keys under 4 bf16 rows 92, read ahead 98, under
    // 4 fp32 rows 95, read ahead 101).  Two steps in turn instead of the copy of one:
    // no faster, and spills.
    constexpr bool EARLY = !MX || (Q32 && !SIDE);
    Step next;
    if (EARLY && t0 < t1) load(t0, next);
    for (int t = t0; t < t1; ++t) {
        const int base = (t < ks.n1 ? t : t - ks.n1 + ks.t_lo) * STEP;
        Step st;
        if constexpr (EARLY) {
            st = next;
            if (t + 1 < t1) load(t + 1, next);
        } else {
            load(t, st);
        }
        const auto& dead = st.dead;
        f32x4 s4[HALVES];
        float vf[FP ? 4 : 1][W];
        uint32_t vw[FP ? 1 : 8][FP ? 1 : W / 2];  // two dims of a key to a word
        if constexpr (FP) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < W; ++x) vf[i][x] = __uint_as_float(st.v[W * i + x]);
            s4[0] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s4[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(st.k[4 * s + e]), qf[s][e], s4[0], 0,
                                                                  0, 0);
        } else {
            bf16x8 kb[HALVES][KS];
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u32x4 w;
                    if constexpr (MX) {
                        const float sc = mx_scale(st.ks[a]);
                        const uint32_t code = st.k[KS * a + s];
                        w = u32x4{mx_decode2<0>(code, sc), mx_decode2<1>(code, sc), mx_decode2<2>(code, sc),
                                  mx_decode2<3>(code, sc)};
                    } else {
#pragma unroll
                        for (int x = 0; x < 4; ++x) w[x] = st.k[4 * (KS * a + s) + x];
                    }
                    kb[a][s] = __builtin_bit_cast(bf16x8, w);
                }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (MX) {
                    const float sc = mx_scale(st.vs[j]);
                    vw[j][0] = mx_decode2<0>(st.v[j], sc);
                    vw[j][1] = mx_decode2<1>(st.v[j], sc);
                    if constexpr (W == 8) {
                        vw[j][2] = mx_decode2<2>(st.v[j], sc);
                        vw[j][3] = mx_decode2<3>(st.v[j], sc);
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < W / 2; ++x) vw[j][x] = st.v[(W / 2) * j + x];
                }
            }
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                s4[a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t3 = QT - 1; t3 >= 0; --t3)
#pragma unroll
                    for (int s = 0; s < KS; ++s)
                        s4[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kb[a][s], qb[t3][s], s4[a], 0, 0, 0);
                if constexpr (SIDE && Q32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s4[a][i] = plus_dpp<kRor8>(plus_dpp<kHalfMirror>(s4[a][i]));
                }
            }
        }

        bool full = base + STEP - 1 <= pmin &&
                    (static_cast<int64_t>(base) > static_cast<int64_t>(pmax) - d.a.window ||
                     base + STEP - 1 < d.a.sinks);
#pragma unroll
        for (int a = 0; a < HALVES; ++a) full = full && !dead[a];
#pragma unroll
        for (int a = 0; a < HALVES; ++a) s4[a] *= d.scale_log2;
        if (!full) {
#pragma unroll
            for (int a = 0; a < HALVES; ++a)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = base + 16 * a + 4 * g + i;
                    s4[a][i] = (dead[a] | !sees(d, vis, key)) ? -INFINITY : s4[a][i];
                    const bool some = !dead[a] & (key < ks.hi) & ((key >= ks.lo) | (key < ks.first));
                    if constexpr (FP) {
#pragma unroll
                        for (int x = 0; x < W; ++x) vf[i][x] = some ? vf[i][x] : 0.0f;
                    } else {
#pragma unroll
                        for (int x = 0; x < W / 2; ++x) vw[4 * a + i][x] = some ? vw[4 * a + i][x] : 0u;
                    }
                }
        }
        float top = fmaxf(fmaxf(s4[0][0], s4[0][1]), fmaxf(s4[0][2], s4[0][3]));
        if constexpr (HALVES == 2)
            top = fmaxf(top, fmaxf(fmaxf(s4[1][0], s4[1][1]), fmaxf(s4[1][2], s4[1][3])));
        top = max_x32(max_x16(top));
        if (__any(top > m)) {
            const float mn = fmaxf(m, top);
            const float f = exp2_fast(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= f;
#pragma unroll
            for (int x = 0; x < W; ++x) acc[x] *= f;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int a = 0; a < HALVES; ++a)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s4[a][i] = exp2_fast(s4[a][i] - ref);
                l += s4[a][i];
            }
        if constexpr (FP) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < W; ++x)
                    acc[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[i][x], s4[0][i], acc[x], 0, 0, 0);
        } else {
            u32x4 pb[PT];  // the weights' terms, 8 bf16 each
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x0 = s4[j / 2][2 * (j & 1)], x1 = s4[j / 2][2 * (j & 1) + 1];
                if constexpr (SIDE) {
                    x0 = less_bits(x0, out1);
                    x1 = less_bits(x1, out1);
                    if constexpr (Q32) {
                        x0 = less_bits(x0, out2);
                        x1 = less_bits(x1, out2);
                    }
                    pb[0][j] = __builtin_amdgcn_perm(__float_as_uint(x1), __float_as_uint(x0), 0x07060302u);
                    continue;
                }
#pragma unroll
                for (int t3 = 0; t3 < PT; ++t3) {
                    pb[t3][j] = pack2_bf16(x0, x1);
                    x0 -= bf16w_lo(pb[t3][j]);
                    x1 -= bf16w_hi(pb[t3][j]);
                }
            }
#pragma unroll
            for (int x = 0; x < W; ++x) {
                u32x4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    w[j] = __builtin_amdgcn_perm(vw[2 * j + 1][x / 2], vw[2 * j][x / 2],
                                                 x & 1 ? 0x07060302u : 0x05040100u);
                const bf16x8 va = __builtin_bit_cast(bf16x8, w);
#pragma unroll
                for (int t3 = PT - 1; t3 >= 0; --t3)
                    acc[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8, pb[t3]), acc[x],
                                                                      0, 0, 0);
            }
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if constexpr (SIDE) {
#pragma unroll
        for (int x = 0; x < W; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (Q32) acc[x][i] = plus_dpp<kHalfMirror>(acc[x][i]);
                acc[x][i] = plus_dpp<kRor8>(acc[x][i]);
            }
    }

    // the wave's part to LDS: row c, dims W (4 g + i) + t
    // (a NaN total is the row's own: scores that it does not see are replaced)
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < W; t += 4) {
            const f32x4 v = {acc[t][i], acc[t + 1][i], acc[t + 2][i], acc[t + 3][i]};
            nan = nan || v[0] != v[0] || v[1] != v[1] || v[2] != v[2] || v[3] != v[3];
            if (c < d.lds_rows) *reinterpret_cast<f32x4*>(o_row(wave, c) + W * (4 * g + i) + t) = v;
        }
    if (g == 0) { sm_m[wave][c] = m; sm_l[wave][c] = l; }
    if (pmin != pmax) {
        const uint64_t bad = __ballot(nan && live && l == l);
        constexpr uint32_t COLUMNS = SIDE ? (1u << side_rows(Q32)) - 1 : 0xFFFFu;
        uint32_t rows = static_cast<uint32_t>(bad | bad >> 16 | bad >> 32 | bad >> 48) & COLUMNS;
        while (rows) {
            const int x = __builtin_ctz(rows);
            rows &= rows - 1;
            const int rr = r0 + x;
            if (!stray<D, KV, STEP>(d, table, h, ks, t0, t1, pmin, pmax, p0 + rr / d.group)) continue;
            redo_row<D, Q32, KV, STEP>(d, table, h, ks, t0, t1, sq.q0 + rr / d.group, h * d.group + rr % d.group,
                                       p0 + rr / d.group, o_row(wave, x), &sm_m[wave][x], &sm_l[wave][x]);
        }
    }
    __syncthreads();

    // join the waves' parts and write the result, or the workgroup's part of it
    constexpr int TPR = D / 8;  // threads of a row, 8 dims each
    for (int x = threadIdx.x; x < kRows * TPR; x += 64 * d.waves) {
        const int dim = 8 * (x % TPR), rc = x / TPR;
        const int rr = r0 + rc;
        if (rr >= nrows) continue;
        float mm = -INFINITY;
        for (int w = 0; w < d.waves; ++w) mm = fmaxf(mm, sm_m[w][rc]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f, o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < d.waves; ++w) {
            const float f = exp2_fast(sm_m[w][rc] - ref);
            ll = fmaf(sm_l[w][rc], f, ll);
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = fmaf(o_row(w, rc)[dim + j], f, o[j]);
        }
        const int head = h * d.group + rr % d.group;
        const int64_t orow = (sq.q0 + rr / d.group) * d.a.q_heads + head;
        if (d.splits > 1) {
            const int64_t slot = d.by_seq ? b * d.max_q + rr / d.group : sq.q0 + rr / d.group;
            const int64_t at = (slot * d.a.q_heads + head) * d.splits + split;
            float* po = d.part + at * D + dim;
            *reinterpret_cast<f32x4*>(po) = f32x4{o[0], o[1], o[2], o[3]};
            *reinterpret_cast<f32x4*>(po + 4) = f32x4{o[4], o[5], o[6], o[7]};
            if (dim == 0) {
                float* ml = d.part + d.slots * d.a.q_heads * d.splits * D + 2 * at;
                ml[0] = mm;
                ml[1] = ll;
            }
        } else {
            const float inv = ll == 0.0f ? 0.0f : __fdiv_rn(1.0f, ll);
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = ll == 0.0f ? 0.0f : o[j] * inv;
            if constexpr (Q32) {
                float* out = static_cast<float*>(d.a.out) + orow * D + dim;
                *reinterpret_cast<f32x4*>(out) = f32x4{o[0], o[1], o[2], o[3]};
                *reinterpret_cast<f32x4*>(out + 4) = f32x4{o[4], o[5], o[6], o[7]};
            } else {
                *reinterpret_cast<u32x4*>(static_cast<bf16_t*>(d.a.out) + orow * D + dim) =
                    u32x4{pack2_bf16(o[0], o[1]), pack2_bf16(o[2], o[3]), pack2_bf16(o[4], o[5]),
                          pack2_bf16(o[6], o[7])};
            }
        }
    }
}

// ---- many rows ----------------------------------------------------------------
//
// The same products on 32 x 32 MFMAs for chunks: a workgroup takes 128 rows (32
// a wave) under one key head and walks 64 keys a step, K and V staged in LDS
// (bf16: global_load_lds straight from the pages; 4 bits: decoded on the way)
// one step ahead in two buffers.
//   S^T = K Q^T     32 keys x 32 rows; a lane holds row lane % 32 and keys
//                   8 (i / 4) + 4 (lane / 32) + i % 4
//   O^T += V^T P^T   32 dims x 32 rows; the 8 weights a lane holds of 16 keys are
//                   the B operand as they are, and V^T comes transposed out of
//                   LDS (ds_read_b64_tr_b16: 4 keys of one dim) in that order.
// The running reference m of a row follows its maximum only when that has grown
// by more than 2^8: weights are then below 256, which neither their bf16 nor the
// fp32 sums feel, and most steps leave the accumulator alone.  With bf16 queries a
// weight is rounded to bf16 for its product with V (half a step, 2^-9, of either
// sign on each of many keys, against 2^-9 in the bf16 output itself; the sum of the
// weights keeps 32 bits): a second term would cost half as many MFMAs again.  fp32
// queries keep three.
// Bound by the matrix cores and what feeds them: 4 x 2048 tokens on 8192 keys, 16
// heads of 128, bf16, 358 to 372 us = 0.88 to 0.91 PFLOP/s (the library's 8192^3
// product 1.16); many times over without a pause 411, at the clock that is left then.  fp32
// queries, three products for one: 858 on a bf16 cache, 874 on 4 bits.
// LDS rows are one key's D values; 16-byte chunks are permuted so that the lanes
// served together (16 keys' same chunk for K, 4 keys' 64 bytes for V) lie in
// different banks.

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 32;            // rows of a wave
constexpr int kBlockRows = kWaves * kTileRows;
constexpr float kLag = 8.0f;

template <int D, bool FP>
__device__ inline int k_swizzle(int key) { return FP || D == 128 ? key & 15 : (key >> 1) & 7; }
template <int D, bool FP>
__device__ inline int v_swizzle(int key) { return FP ? 0 : D == 128 ? (key & 3) << 2 : ((key >> 1) & 1) << 2; }

#define APS_AGP(p) ((const __attribute__((address_space(1))) void*)(p))
#define APS_ALP(p) ((__attribute__((address_space(3))) void*)(p))

template <int D, bool Q32, Kv KV>
__global__ void __launch_bounds__(64 * kWaves, 2)
k_paged_tiles(PagedDev d) {
    constexpr int BLOCK = kBlockRows;
    constexpr bool FP = KV == Kv::kF32;
    constexpr int KEYS = FP ? 32 : 64;         // keys of a step
    constexpr int U = KEYS / 32;               // 32-key halves of it
    constexpr int GROUPS = KEYS / 16;          // 16-key groups, each of one page
    constexpr int ROW = (FP ? 4 : 2) * D;      // LDS bytes of a key
    constexpr int CH = ROW / 16;               // 16-byte chunks of a key
    constexpr int QT = Q32 ? 3 : 1, PT = Q32 ? 3 : 1;
    constexpr int KS = D / (FP ? 8 : 16);      // chunks of a lane: its half of a key's dims
    constexpr int DT = D / 32;
    __shared__ __align__(1024) uint8_t sm[2][2][KEYS * ROW];  // [k, v][buffer]

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, c = lane & 31, hf = lane >> 5;
    // Workgroups take the row blocks that there are, sequence by sequence, so
    // that those without one are the last of the grid (left between, they
    // take their XCD's share: 3 ragged chunks of 500 tokens on a 4-bit cache, with
    // the join, 69 us, closed up 55).  Row blocks of one key head go round the
    // XCDs: each L2 reads every sequence's keys, but no XCD is left with the long
    // ones.
    uint32_t id = blockIdx.x;
    const uint32_t per = static_cast<uint32_t>(d.c.kv_heads * d.splits);
    int64_t b = -1;
    uint32_t row_blocks = 0;
    for (int64_t b0 = 0; b0 < d.a.batch; b0 += 64) {
        uint32_t n = 0;
        if (b0 + lane < d.a.batch) {
            const Seq one = clipped(d, d.a.q_offsets[b0 + lane], d.a.q_offsets[b0 + lane + 1], 0);
            n = static_cast<uint32_t>((rows_of(d, one.len) + BLOCK - 1) / BLOCK);
        }
        uint32_t upto = n;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) {
            const uint32_t v = __shfl_up(upto, x);
            upto += lane >= x ? v : 0u;
        }
        const uint64_t past = __ballot(id < upto * per);
        if (past) {
            const int at = __builtin_ctzll(past);
            row_blocks = __builtin_amdgcn_readlane(n, at);
            id -= (__builtin_amdgcn_readlane(upto, at) - row_blocks) * per;
            b = b0 + at;
            break;
        }
        id -= __builtin_amdgcn_readlane(upto, 63) * per;
    }
    if (b < 0) return;
    const int split = __builtin_amdgcn_readfirstlane(id % d.splits);
    id /= d.splits;
    // the last rows see the most keys: they start first
    const int rb = __builtin_amdgcn_readfirstlane(row_blocks - 1 - id % row_blocks);
    const int h = __builtin_amdgcn_readfirstlane(id / row_blocks);
    const Seq sq = sequence(d, b);
    const int nrows = rows_of(d, sq.len);
    const int rb0 = rb * BLOCK;
    const int32_t* table = d.a.page_table + b * d.a.table_stride;
    const int p0 = sq.kv - sq.len;
    const int rb1 = (rb0 + BLOCK < nrows ? rb0 + BLOCK : nrows) - 1;
    const Keys ks = visible<KEYS>(d, p0 + rb0 / d.group, p0 + rb1 / d.group);
    const int each = __builtin_amdgcn_readfirstlane((ks.steps + d.splits - 1) / d.splits);
    const int t0 = split * each < ks.steps ? split * each : ks.steps;
    const int t1 = t0 + each < ks.steps ? t0 + each : ks.steps;

    const int r0 = rb0 + wave * kTileRows;
    const bool any = r0 < nrows;
    const int r_last = r0 + kTileRows - 1 < nrows ? r0 + kTileRows - 1 : nrows - 1;
    const int pmin = __builtin_amdgcn_readfirstlane(p0 + r0 / d.group);
    const int pmax = __builtin_amdgcn_readfirstlane(any ? p0 + r_last / d.group : -1);
    const int row = r0 + c;
    const bool live = row < nrows;
    const int tok = live ? row / d.group : 0, qh = h * d.group + (live ? row % d.group : 0);
    const View vis = view(d, live ? p0 + tok : -1);

    // ---- staging, one step ahead.  64 keys: a wave copies 16 keys of K and of V;
    // 32 keys: two waves copy K, two V.
    const int grp = wave % GROUPS;
    const bool with_k = GROUPS == kWaves || wave < GROUPS, with_v = GROUPS == kWaves || wave >= GROUPS;
    auto base_of = [&](int t) { return (t < ks.n1 ? t : t - ks.n1 + ks.t_lo) * KEYS; };
    u32x4 mk{}, mv{};
    uint32_t mks = 0, mvs = 0;
    int pages = -1;          // lane GROUPS i + a: the page of 16 keys a of step i of 64 / GROUPS
    uint32_t dead_next = 0;  // bit a: 16 keys a of the step that was fetched have no page
    // where a lane's 16 bytes of each copy come from, past the (uniform) place of
    // the 16 keys: 32-bit offsets, one add in the load (4 bits: four lanes a key,
    // codes and scales)
    constexpr bool MX = KV == Kv::kMx;
    constexpr int RPI = MX ? 16 : 1024 / ROW;  // keys of one copy
    uint32_t k_src[16 / RPI], v_src[16 / RPI];
#pragma unroll
    for (int i = 0; i < 16 / RPI; ++i) {
        const int r = RPI * i + lane / CH;
        k_src[i] = MX ? lane / 4 * (D / 2) + (lane & 3) * (D / 8) : r * ROW + 16 * ((lane % CH) ^ k_swizzle<D, FP>(r));
        v_src[i] = MX ? lane / 4 * (D / 32) + (lane & 3) * (D / 4) / 32
                      : r * ROW + 16 * ((lane % CH) ^ v_swizzle<D, FP>(r));
    }
    auto fetch1 = [&](int which, int64_t hrow, int buf) {  // one operand's 16 keys, to LDS or (4 bits) to registers
        const uint8_t* src = static_cast<const uint8_t*>(which ? d.c.v : d.c.k);
        if constexpr (KV != Kv::kMx) {
            src += hrow * ROW;
#pragma unroll
            for (int i = 0; i < 16 / RPI; ++i)
                __builtin_amdgcn_global_load_lds(APS_AGP(src + (which ? v_src : k_src)[i]),
                                                 APS_ALP(&sm[which][buf][(16 * grp + RPI * i) * ROW]), 16, 0, 0);
        } else {
            src += hrow * (D / 2);
            u32x4& w = which ? mv : mk;
            if constexpr (D == 128) {
                w = *reinterpret_cast<const u32x4*>(src + k_src[0]);
            } else {
                const u32x2 half = *reinterpret_cast<const u32x2*>(src + k_src[0]);
                w = u32x4{half[0], half[1], 0u, 0u};
            }
            const uint8_t* sc = (which ? d.c.v_scale : d.c.k_scale) + hrow * (D / 32);
            (which ? mvs : mks) = sc[v_src[0]];
        }
    };
    auto fetch = [&](int t, int buf) {
        const int slot = (t - t0) % (64 / GROUPS);
        if (slot == 0) pages = page_of<KEYS>(d, table, ks, t + lane / GROUPS, t1, lane % GROUPS);
        dead_next = static_cast<uint32_t>(__ballot(pages < 0) >> (GROUPS * slot)) & ((1u << GROUPS) - 1);
        const int page = __builtin_amdgcn_readlane(pages, GROUPS * slot + grp);
        const int64_t hrow = ((static_cast<int64_t>(page < 0 ? 0 : page) * d.c.kv_heads + h) << d.page_shift) +
                             ((base_of(t) + 16 * grp) & ((1 << d.page_shift) - 1));
        if (with_k) fetch1(0, hrow, buf);
        if (with_v) fetch1(1, hrow, buf);
    };
    auto decode1 = [&](int which, int buf) {
        const int r = lane / 4;
        const u32x4 w = which ? mv : mk;
        const float sc = mx_scale(which ? mvs : mks);
        uint8_t* at = &sm[which][buf][(16 * grp + r) * ROW];
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const int chunk = ((lane & 3) * (D / 32) + j) ^ (which ? v_swizzle<D, FP>(r) : k_swizzle<D, FP>(r));
            *reinterpret_cast<u32x4*>(at + 16 * chunk) = u32x4{mx_decode2<0>(w[j], sc), mx_decode2<1>(w[j], sc),
                                                               mx_decode2<2>(w[j], sc), mx_decode2<3>(w[j], sc)};
        }
    };
    auto commit = [&](int t, int buf) {
        if constexpr (KV == Kv::kMx) {
            if (with_k) decode1(0, buf);
            if (with_v) decode1(1, buf);
        } else {
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's copies are in LDS
        }
        // values that no row of the block sees become zeros
        const int key0 = base_of(t) + 16 * grp;
        const bool gone = dead_next >> grp & 1u;
        const bool whole = !gone && key0 + 15 < ks.hi && (key0 >= ks.lo || key0 + 15 < ks.first);
        if (with_v && !whole) {
            const int r = lane / 4, key = key0 + r;
            if (gone || key >= ks.hi || (key < ks.lo && key >= ks.first)) {
                u32x4* at = reinterpret_cast<u32x4*>(&sm[1][buf][(16 * grp + r) * ROW + (lane & 3) * (ROW / 4)]);
#pragma unroll
                for (int j = 0; j < ROW / 64; ++j) at[j] = u32x4{0u, 0u, 0u, 0u};
            }
        }
    };

    if (t0 < t1) fetch(t0, 0);  // on its way while the queries are read

    // queries: a lane holds dims 16 s + 8 hf + j of its row; the sign of the
    // scale goes into them (exactly), so that the largest product is the largest
    // score, and of a scale of 0 the zero, or NaN where they are not finite
    bf16x8 qb[FP ? 1 : QT][FP ? 1 : KS];
    f32x4 qf[FP ? KS : 1];
    const float cs = d.scale_log2 == 0.0f ? 1.0f : fabsf(d.scale_log2);
    const float qs = d.scale_log2 < 0.0f ? -1.0f : d.scale_log2 == 0.0f ? 0.0f : 1.0f;
    {
        const int64_t qat = (sq.q0 + tok) * d.a.q_stride + static_cast<int64_t>(qh) * D;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int dim = (FP ? 8 : 16) * s + (FP ? 4 : 8) * hf;
            if constexpr (FP) {
                qf[s] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(d.a.q) + qat + dim) * qs;
                continue;
            }
            if constexpr (FP) {
            } else if constexpr (Q32) {
                const float* p = static_cast<const float*>(d.a.q) + qat + dim;
                const f32x4 x0 = *reinterpret_cast<const f32x4*>(p), x1 = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float x = (j < 4 ? x0[j & 3] : x1[j & 3]) * qs;
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        const float hi = bf16_round(x);
                        qb[t][s][j] = static_cast<__bf16>(hi);
                        x -= hi;
                    }
                }
            } else {
                u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const bf16_t*>(d.a.q) + qat + dim);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = pack2_bf16(bf16w_lo(w[j]) * qs, bf16w_hi(w[j]) * qs);
                qb[0][s] = __builtin_bit_cast(bf16x8, w);
            }
        }
    }

    // LDS offsets of a lane's operands
    int k_off[KS], v_off[DT];
#pragma unroll
    for (int s = 0; s < KS; ++s) k_off[s] = c * ROW + (((2 * s + hf) ^ k_swizzle<D, FP>(c)) << 4);
    {
        const int i = lane & 15, r = i >> 2, dh = (lane >> 4) & 1;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            v_off[t] = (4 * hf + r) * ROW + (((4 * t + 2 * dh + ((i & 3) >> 1)) ^ v_swizzle<D, FP>(r)) << 4) + 8 * (i & 1);
    }

    f32x16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    if (t0 < t1) commit(t0, 0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1, base = base_of(t);
        const uint32_t dead = dead_next;
        if (t + 1 < t1) fetch(t + 1, buf ^ 1);
        // a step that no row of this wave sees is left out
        const bool none = base > pmax ||
                          (static_cast<int64_t>(base) + KEYS - 1 <= static_cast<int64_t>(pmin) - d.a.window &&
                           base >= d.a.sinks);
        if (!none) {
            const uint8_t* kt = sm[0][buf];
            const uint8_t* vt = sm[1][buf];
            f32x16 s[U];
            // the other wave of the SIMD does its softmax meanwhile (391 -> 378 us at 4 x
            // 2048 tokens on 8192 keys; with the second product too, no gain)
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
#pragma unroll
                for (int x = 0; x < KS; ++x) {
                    if constexpr (FP) {
                        const f32x4 kf = *reinterpret_cast<const f32x4*>(kt + k_off[x]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], qf[x][j], s[u], 0, 0, 0);
                    } else {
                        const bf16x8 kf = *reinterpret_cast<const bf16x8*>(kt + k_off[x] + u * 32 * ROW);
#pragma unroll
                        for (int q3 = QT - 1; q3 >= 0; --q3)
                            s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qb[q3][x], s[u], 0, 0, 0);
                    }
                }
            }
            __builtin_amdgcn_s_setprio(0);
            const bool full = dead == 0 && base + KEYS - 1 <= pmin &&
                              (static_cast<int64_t>(base) > static_cast<int64_t>(pmax) - d.a.window ||
                               base + KEYS - 1 < d.a.sinks);
            if (!full) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int at = 32 * u + 8 * (i / 4) + 4 * hf + i % 4;
                        const bool out = (dead >> (2 * u + i / 8) & 1u) | !sees(d, vis, base + at);
                        s[u][i] = out ? -INFINITY : s[u][i];
                    }
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(fmaxf(top, s[0][i]), s[U - 1][i]);
            top = max_x32(top) * cs;
            if (__any(top > m + kLag)) {
                const float mn = top > m + kLag ? top : m;
                const float f = exp2_fast(m - (mn == -INFINITY ? 0.0f : mn));
                m = mn;
                l *= f;
#pragma unroll
                for (int x = 0; x < DT; ++x) acc[x] *= f;
            }
            const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[u][i] = exp2_fast(fmaf(s[u][i], cs, -ref));
                    l += s[u][i];
                }
            if constexpr (FP) {
                // key 8 (i / 4) + 4 hf + i % 4 of V, dims DT c .. DT c + DT - 1
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint8_t* at = vt + (8 * (i / 4) + 4 * hf + i % 4) * ROW + 4 * DT * c;
                    float v[DT];
                    if constexpr (DT == 4) {
                        const f32x4 w = *reinterpret_cast<const f32x4*>(at);
#pragma unroll
                        for (int y = 0; y < 4; ++y) v[y] = w[y];
                    } else {
                        const u32x2 w = *reinterpret_cast<const u32x2*>(at);
                        v[0] = __uint_as_float(w[0]);
                        v[1] = __uint_as_float(w[1]);
                    }
#pragma unroll
                    for (int y = 0; y < DT; ++y)
                        acc[y] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[y], s[0][i], acc[y], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int x = 0; x < 4; ++x) {   // 16 keys each
                    u32x4 pb[PT];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float a0 = s[x / 2][8 * (x & 1) + 2 * j], a1 = s[x / 2][8 * (x & 1) + 2 * j + 1];
#pragma unroll
                        for (int p3 = 0; p3 < PT; ++p3) {
                            pb[p3][j] = pack2_bf16(a0, a1);
                            a0 -= bf16w_lo(pb[p3][j]);
                            a1 -= bf16w_hi(pb[p3][j]);
                        }
                    }
#pragma unroll
                    for (int y = 0; y < DT; ++y) {
                        typedef __attribute__((address_space(3))) s16x4* lds_s4;
                        const uint8_t* at = vt + v_off[y] + 16 * x * ROW;
                        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at));
                        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at + 8 * ROW));
                        const u32x2 wl = __builtin_bit_cast(u32x2, lo), wh = __builtin_bit_cast(u32x2, hi);
                        const bf16x8 va = __builtin_bit_cast(bf16x8, u32x4{wl[0], wl[1], wh[0], wh[1]});
#pragma unroll
                        for (int p3 = PT - 1; p3 >= 0; --p3)
                            acc[y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, __builtin_bit_cast(bf16x8, pb[p3]), acc[y],
                                                                              0, 0, 0);
                    }
                }
            }
        }
        if (t + 1 < t1) commit(t + 1, buf ^ 1);
        __syncthreads();
    }
    l += __shfl_xor(l, 32);

    // the dim that a lane holds in acc[y][i]
    auto dim_of = [&](int y, int i) {
        const int m = 8 * (i / 4) + 4 * hf + i % 4;
        return FP ? DT * m + y : 32 * y + m;
    };
    bool nan = false;  // a NaN total is the row's own: scores that it does not see are replaced
#pragma unroll
    for (int y = 0; y < DT; ++y)
#pragma unroll
        for (int i = 0; i < 16; ++i) nan = nan || acc[y][i] != acc[y][i];
    const uint64_t bad = __ballot(nan && live && l == l);
    uint32_t rows = static_cast<uint32_t>(bad | bad >> 32);
    // (values are set to zero where no row of the block sees them: a wave's rows may
    // all be one token's that does not see what another wave's do)
    if (any && rb0 / d.group != rb1 / d.group) {
        // every wave is past the last step's barrier: the staging buffers are free
        float* red = reinterpret_cast<float*>(&sm[0][0][0]) + wave * (D + 2);
        while (rows) {
            const int x = __builtin_ctz(rows);
            rows &= rows - 1;
            const int rr = r0 + x;
            if (!stray<D, KV, KEYS>(d, table, h, ks, t0, t1, pmin, pmax, p0 + rr / d.group)) continue;
            redo_row<D, Q32, KV, KEYS>(d, table, h, ks, t0, t1, sq.q0 + rr / d.group,
                                            h * d.group + rr % d.group, p0 + rr / d.group, red, red + D, red + D + 1);
            __builtin_amdgcn_wave_barrier();
            if (c == x) {
                m = red[D];
                l = red[D + 1];
#pragma unroll
                for (int y = 0; y < DT; ++y)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[y][i] = red[dim_of(y, i)];
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
    if (!live) return;
    const int64_t orow = (sq.q0 + tok) * d.a.q_heads + qh;
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    const int64_t at = orow * d.splits + split;
    if (d.splits > 1 && hf == 0) {
        float* ml = d.part + d.slots * d.a.q_heads * d.splits * D + 2 * at;
        ml[0] = m;
        ml[1] = l;
    }
    if constexpr (FP) {
        float* to = d.splits > 1 ? d.part + at * D : static_cast<float*>(d.a.out) + orow * D;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v[DT];
#pragma unroll
            for (int y = 0; y < DT; ++y)
                v[y] = d.splits > 1 ? acc[y][i] : l == 0.0f ? 0.0f : acc[y][i] * inv;
            if constexpr (DT == 4) *reinterpret_cast<f32x4*>(to + dim_of(0, i)) = f32x4{v[0], v[1], v[2], v[3]};
            else *reinterpret_cast<u32x2*>(to + dim_of(0, i)) = u32x2{__float_as_uint(v[0]), __float_as_uint(v[1])};
        }
        return;
    }
#pragma unroll
    for (int y = 0; y < DT; ++y)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int dim = 32 * y + 2 * i + 4 * hf;
            f32x4 v = {acc[y][i], acc[y][i + 1], acc[y][i + 2], acc[y][i + 3]};
            if (d.splits > 1) {
                *reinterpret_cast<f32x4*>(d.part + at * D + dim) = v;
                continue;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = l == 0.0f ? 0.0f : v[j] * inv;
            if constexpr (Q32)
                *reinterpret_cast<f32x4*>(static_cast<float*>(d.a.out) + orow * D + dim) = v;
            else
                *reinterpret_cast<u32x2*>(static_cast<bf16_t*>(d.a.out) + orow * D + dim) =
                    u32x2{pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3])};
        }
}

// out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s over the splits of one
// (row, head), a workgroup each.  The row's sequence is looked up, 64 at a time,
// while its parts are on their way (by_seq: it is known): rows that no sequence
// of this launch names are left as they were.
template <int D, bool Q32, int JW>
__global__ void __launch_bounds__(64 * JW)
k_paged_join(PagedDev d) {
    constexpr int PER = D / 64;
    __shared__ float part[JW][D];
    __shared__ float weight[JW][JW == 1 ? 1 : kMaxSplits];  // a wave's own copy
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t at = static_cast<int64_t>(blockIdx.x) * d.splits;
    const uint32_t slot = blockIdx.x / static_cast<uint32_t>(d.a.q_heads);
    const int head = static_cast<int>(blockIdx.x - slot * static_cast<uint32_t>(d.a.q_heads));
    int64_t row = slot;
    const float* ml = d.part + d.slots * d.a.q_heads * d.splits * D + 2 * at;
    const float* po = d.part + at * D + PER * lane;
    constexpr int MOST = JW == 1 ? kFewSplits : kMaxSplits, MX = (MOST + 63) / 64;
    // few splits: everything is on its way before the first wait
    float few[JW == 1 ? kFewSplits : 1][PER];
    if constexpr (JW == 1) {
#pragma unroll
        for (int s = 0; s < kFewSplits; ++s)
            if (s < d.splits) {
#pragma unroll
                for (int j = 0; j < PER; ++j) few[s][j] = po[static_cast<int64_t>(s) * D + j];
            }
    }
    float m[MX], l[MX], top = -INFINITY;
#pragma unroll
    for (int x = 0; x < MX; ++x) {
        const int s = 64 * x + lane;
        m[x] = s < d.splits ? ml[2 * s] : -INFINITY;
        l[x] = s < d.splits ? ml[2 * s + 1] : 0.0f;
        top = fmaxf(top, m[x]);
    }
    bool named = false;
    if (d.by_seq) {
        const uint32_t b = slot / static_cast<uint32_t>(d.max_q), tok = slot - b * static_cast<uint32_t>(d.max_q);
        const Seq one = sequence(d, b);
        row = one.q0 + tok;
        named = static_cast<int64_t>(tok) * d.group < rows_of(d, one.len);
    }
    for (int64_t b0 = 0; b0 < d.a.batch && !named && !d.by_seq; b0 += 64) {
        bool mine = false;
        if (b0 + lane < d.a.batch) {
            const Seq one = clipped(d, d.a.q_offsets[b0 + lane], d.a.q_offsets[b0 + lane + 1], 0);
            mine = row >= one.q0 && (row - one.q0) * d.group < rows_of(d, one.len);
        }
        named = __ballot(mine) != 0;
    }
    if (!named) return;
    const int64_t orow = row * d.a.q_heads + head;
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, w[MX];
#pragma unroll
    for (int x = 0; x < MX; ++x) {
        w[x] = exp2_fast(m[x] - ref);
        sum = fmaf(w[x], l[x], sum);
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x);
    float o[PER] = {};
    if constexpr (JW == 1) {
#pragma unroll
        for (int s = 0; s < kFewSplits; ++s)
            if (s < d.splits) {
                const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w[0]), s));
#pragma unroll
                for (int j = 0; j < PER; ++j) o[j] = fmaf(ws, few[s][j], o[j]);
            }
    } else {
#pragma unroll
        for (int x = 0; x < MX; ++x) weight[wave][64 * x + lane] = w[x];
        __builtin_amdgcn_wave_barrier();
#pragma unroll 4
        for (int s = wave; s < d.splits; s += JW) {
            const float ws = weight[wave][s];
#pragma unroll
            for (int j = 0; j < PER; ++j) o[j] = fmaf(ws, po[static_cast<int64_t>(s) * D + j], o[j]);
        }
    }
    if constexpr (JW > 1) {
#pragma unroll
        for (int j = 0; j < PER; ++j) part[wave][PER * lane + j] = o[j];
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int x = 1; x < JW; ++x)
#pragma unroll
            for (int j = 0; j < PER; ++j) o[j] += part[x][PER * lane + j];
    }
    const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const float v = sum == 0.0f ? 0.0f : o[j] * inv;
        if constexpr (Q32) static_cast<float*>(d.a.out)[orow * D + PER * lane + j] = v;
        else static_cast<bf16_t*>(d.a.out)[orow * D + PER * lane + j] = static_cast<bf16_t>(pack2_bf16(v, 0.0f) & 0xFFFFu);
    }
}

// One launch over the sequences of least .. most rows under a key head; `beside`:
// the short ones next to one that is not.
PagedDev plan_one(const KvCache& c, const PagedArgs& a, int64_t least, int64_t most, bool beside) {
    PagedDev d;
    d.a = a;
    d.c = c;
    d.page_shift = c.page_shift;
    d.group = a.q_heads / c.kv_heads;
    d.scale_log2 = a.scale * kLog2e;
    d.least = static_cast<int>(least);
    d.most = static_cast<int>(most);
    d.max_q = std::min<int64_t>(a.max_q_len, std::max<int64_t>(most / d.group, 1));
    const int64_t rows = d.max_q * d.group, heads = a.batch * c.kv_heads;
    // keys one tile can see, in steps of 32
    const int64_t keys = std::min<int64_t>(a.max_kv_len, static_cast<int64_t>(a.window) + a.sinks + 16);
    const int64_t steps = ceil_div(keys, 32);
    d.tiled = most >= kTiledRows;
    d.waves = kWaves;
    d.lds_rows = static_cast<int>(std::min<int64_t>(kRows, rows));
    d.row_tiles = static_cast<int>(ceil_div(rows, d.tiled ? kBlockRows : kRows));
    int64_t tiles = heads * d.row_tiles, splits;
    if (d.tiled) {
        // the blocks of rows that there can be, and about how many there are; two
        // workgroups a CU and no more (a third round costs what a split saves)
        tiles = std::min<int64_t>(tiles, c.kv_heads * (a.rows * d.group / kBlockRows + a.batch));
        // (short ones beside them taken for steps of a token)
        const int64_t long_rows = least > 1 ? std::max<int64_t>(a.rows - a.batch, 1) : a.rows;
        const int64_t about = std::max<int64_t>(ceil_div(long_rows * a.q_heads, kBlockRows),
                                                c.kv_heads * (least > 1 ? 1 : a.batch));
        splits = std::min<int64_t>(512 / about, ceil_div(steps, 8));
    } else {
        // four workgroups a CU of a large batch, two where there are few tiles and
        // the parts to join weigh more (us with two / four: 64 x 8192 keys 148 /
        // 145, in 4 bits 99 / 89; 32 x 2051 27 / 31, 1 x 100000 39 / 42)
        // (beside chunks: what there is when all but one are steps of a token, not the
        // two tiles that each could have)
        const int64_t about = beside ? (a.batch - 1) * c.kv_heads * ceil_div(d.group, kRows) : tiles;
        splits = std::min<int64_t>(ceil_div(about > 128 ? 1024 : 512, about), ceil_div(steps, 2 * kWaves));
        if (splits > 1 && steps <= 4 * kMostWaves && kMostWaves * d.lds_rows * (c.head_dim + 4) * 4 <= kPlainLds) {
            // short: one larger workgroup instead of a second launch
            d.waves = kMostWaves;
            splits = 1;
        }
    }
    d.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(splits, kMaxSplits)));
    d.blocks = tiles * d.splits;
    // the short sequences of a batch with chunks have few of its rows
    d.by_seq = !d.tiled && a.batch * d.max_q < a.rows;
    d.slots = d.by_seq ? a.batch * d.max_q : a.rows;
    return d;
}

int64_t part_floats(const PagedDev& d) {
    return d.splits > 1 ? ceil_div(d.slots * d.a.q_heads * d.splits * (d.c.head_dim + 2), 64) * 64 : 0;
}

// The launches of a call: sequences of kTiledRows rows and more to k_paged_tiles,
// shorter ones to k_paged_rows, by each one's own rows, so that the bits of its
// weights are not its neighbours' choice.  Which is which stands on the device; the
// host launches both unless the sizes leave no room for one kind: max_q_len is
// short itself, or the rows are too many for a short one beside batch - 1 of
// max_q_len.  (bf16, 16 heads of 128, us as one launch of k_paged_tiles / as two:
// 4 prompts of 512 and 60 steps on 8192 keys 296 / 359, one of the steps on 100000
// 2403 / 547; 2 prompts and 62 steps 267 / 294, in 4 bits 225 / 177.  Where all are
// prompts, 16 of up to 512, the launch for none costs 3 of 41.)
struct Plan {
    PagedDev d[2];
    int n;
};
Plan plan(const KvCache& c, const PagedArgs& a) {
    Plan p;
    const int64_t group = a.q_heads / c.kv_heads, longest = a.max_q_len * group, few = (kTiledRows - 1) / group;
    const bool both = longest >= kTiledRows && few > 0 && a.rows <= (a.batch - 1) * a.max_q_len + few;
    p.n = both ? 2 : 1;
    p.d[0] = plan_one(c, a, both ? kTiledRows : 1, longest, false);
    if (both) p.d[1] = plan_one(c, a, 1, kTiledRows - 1, true);
    return p;
}

// The waves that join a row's parts.
// (us of the call with a wave a row / four: 16 x 8192 keys, 8 parts, 45.5 / 46.4;
// with four / sixteen: 1 x 131072, 128 parts, 47.6 / 47.0, 1 x 20000, 79 parts,
// 16.5 / 15.9)
int join_waves(const PagedDev& d) { return d.splits > 64 ? 16 : d.splits > kFewSplits ? 4 : 1; }

template <int D, bool Q32, Kv KV>
hipError_t launch(const PagedDev& d, hipStream_t s) {
    const dim3 blocks(static_cast<unsigned>(d.blocks)), grid(static_cast<unsigned>(d.slots * d.a.q_heads));
    if (d.tiled)
        hipLaunchKernelGGL((k_paged_tiles<D, Q32, KV>), blocks, dim3(64 * kWaves), 0, s, d);
    else if (KV != Kv::kF32 && d.lds_rows <= side_rows(Q32))
        hipLaunchKernelGGL((k_paged_rows<D, Q32, KV, KV != Kv::kF32>), blocks, dim3(64 * d.waves),
                           static_cast<unsigned>(d.waves) * d.lds_rows * (D + 4) * 4, s, d);
    else
        hipLaunchKernelGGL((k_paged_rows<D, Q32, KV, false>), blocks, dim3(64 * d.waves),
                           static_cast<unsigned>(d.waves) * d.lds_rows * (D + 4) * 4, s, d);
    if (d.splits > 1 && join_waves(d) == 16) hipLaunchKernelGGL((k_paged_join<D, Q32, 16>), grid, dim3(1024), 0, s, d);
    else if (d.splits > 1 && join_waves(d) == 4) hipLaunchKernelGGL((k_paged_join<D, Q32, 4>), grid, dim3(256), 0, s, d);
    else if (d.splits > 1) hipLaunchKernelGGL((k_paged_join<D, Q32, 1>), grid, dim3(64), 0, s, d);
    return hipGetLastError();
}

template <int D>
hipError_t launch_d(const PagedDev& d, bool q_f32, hipStream_t s) {
    if (d.c.type == Kv::kF32) return launch<D, true, Kv::kF32>(d, s);
    if (d.c.type == Kv::kBf16)
        return q_f32 ? launch<D, true, Kv::kBf16>(d, s) : launch<D, false, Kv::kBf16>(d, s);
    return q_f32 ? launch<D, true, Kv::kMx>(d, s) : launch<D, false, Kv::kMx>(d, s);
}

}  // namespace

int64_t attention_paged_threads(const KvCache& cache, const PagedArgs& a) {
    const Plan p = plan(cache, a);
    int64_t n = 0;
    for (int i = 0; i < p.n; ++i) {
        const PagedDev& d = p.d[i];
        n = std::max({n, d.blocks * 64 * (d.tiled ? kWaves : d.waves), d.splits > 1 ? d.slots * a.q_heads * 64 * join_waves(d) : 0});
    }
    return n;
}

size_t attention_paged_part_bytes(const KvCache& cache, const PagedArgs& a) {
    const Plan p = plan(cache, a);
    int64_t n = 0;
    for (int i = 0; i < p.n; ++i) n += part_floats(p.d[i]);
    return static_cast<size_t>(n) * 4;
}

hipError_t launch_attention_paged(const KvCache& cache, const PagedArgs& a, bool q_f32, hipStream_t s) {
    if (a.rows <= 0 || a.batch <= 0 || a.max_q_len <= 0) return hipSuccess;
    Plan p = plan(cache, a);
    float* part = a.part;
    for (int i = 0; i < p.n; ++i) {
        p.d[i].part = part;
        part += part_floats(p.d[i]);
        const hipError_t e = cache.head_dim == 128 ? launch_d<128>(p.d[i], q_f32, s) : launch_d<64>(p.d[i], q_f32, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace aps
