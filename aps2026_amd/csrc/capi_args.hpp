// Checks of arguments that the serving operators' C entry points share.
#pragma once

#include "../../include/aps_moe.h"
#include "common.hpp"

namespace aps {
namespace args {

constexpr int64_t kMaxRows = int64_t(1) << 30;

inline bool mis(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

inline bool overlap(const void* p, size_t np, const void* q, size_t nq) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return np && nq && a < b + nq && b < a + np;
}

// `count` rows of `width` bytes, `stride` bytes apart.
typedef __int128 wide;
struct Rows {
    const void* at;
    int64_t count, width;
    wide stride;
};
inline Rows rows_of(const void* p, int64_t rows, int64_t values, int64_t stride, uintptr_t elt) {
    const int64_t e = static_cast<int64_t>(elt);
    return {p, p ? rows : 0, values * e, static_cast<wide>(stride) * e};
}
// True if a row of a shares a byte with a row of b: of slices of one wider row,
// which lie between each other, none does.
inline bool overlap(const Rows& a, const Rows& b) {
    if (a.count <= 0 || b.count <= 0 || a.width <= 0 || b.width <= 0) return false;
    const wide d = static_cast<wide>(reinterpret_cast<uintptr_t>(b.at)) - reinterpret_cast<uintptr_t>(a.at);
    if (d >= (a.count - 1) * a.stride + a.width ||
        -d >= (b.count - 1) * b.stride + b.width)
        return false;
    if (a.count == 1 && b.count == 1) return true;
    auto floor_div = [](wide x, wide y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
    // the first row of b that ends behind the start of a's row i, from
    // b.width + d + j stride > i stride; rows of one stride are alike for all i
    if (a.stride == b.stride || a.count == 1 || b.count == 1) {
        // (a single row's stride is the other's)
        const wide s = a.count == 1 ? b.stride : a.stride;
        const wide first = -(a.count - 1), last = b.count - 1;
        wide j = floor_div(-d - b.width, s) + 1;
        if (j < first) j = first;
        return j <= last && d + j * s < a.width;
    }
    for (int64_t i = 0; i < a.count; ++i) {
        const wide to = i * a.stride;
        wide j = floor_div(to - d - b.width, b.stride) + 1;
        if (j < 0) j = 0;
        if (j < b.count && d + j * b.stride < to + a.width) return true;
    }
    return false;
}

inline int launched(hipError_t err, const char* what) {
    if (err == hipSuccess) return APS_OK;
    return fail(APS_ERR_HIP, "%s: %s", what, hipGetErrorString(err));
}

}  // namespace args
}  // namespace aps
