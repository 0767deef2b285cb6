// Whether tensors of a call share memory, on the host: an output that lies over an input or another output at an offset
// is a race between the workgroups that read the one and write the other.
//
// A tensor of heads is a set of equal runs of bytes, at + i * row + h * head for i < rows and h < heads. Views that
// interleave (q, k and v in one tensor) have spans that overlap and share nothing, so that the runs themselves are compared:
// exactly, unless that would take more than kMostSteps steps (strides that have nothing to do with each other, and no run
// found that is shared); such a call counts as one that shares.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <numeric>

#include "trellis_sparse.h"

namespace tsp {

// Whether [a, a + an) and [b, b + bn) share a byte.
inline bool overlap(const void* a, size_t an, const void* b, size_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && an && bn && x < y + bn && y < x + an;
}

struct Runs {
    int64_t at, rows, row, heads, head, width;      // bytes; none where width or rows is 0
    int64_t span() const { return (rows - 1) * row + (heads - 1) * head + width; }
};
inline Runs runs_of(const void* p, int64_t bytes) { return Runs{(int64_t)reinterpret_cast<uintptr_t>(p), p ? 1 : 0, 0, 1, 0, bytes}; }
// n rows of heads of d elements of `size` bytes. Runs that touch become one.
inline Runs runs_of(const tsp_heads& t, int64_t n, int heads, int d, size_t size) {
    Runs r = runs_of(t.data, d * (int64_t)size);
    r.rows = n, r.row = t.row_stride * (int64_t)size, r.heads = heads, r.head = t.head_stride * (int64_t)size;
    for (int i = 0; i < 2; ++i) {       // (whichever of the two is inside the other)
        if (r.heads > 1 && r.head <= r.width) r.width += (r.heads - 1) * r.head, r.heads = 1;
        if (r.rows > 1 && r.row <= r.width) r.width += (r.rows - 1) * r.row, r.rows = 1;
    }
    return r;
}

// Whether run b, which begins `from` + k * step bytes after run a, shares a byte with it for some k in [lo, hi].
inline bool steps_meet(int64_t from, int64_t step, int64_t lo, int64_t hi, int64_t a_width, int64_t b_width) {
    if (step == 0) return lo <= hi && from < a_width && from + b_width > 0;
    const int64_t below = -b_width - from;      // k * step > below; the least such k, and lo
    const int64_t q = below / step, k = std::max(lo, q - (below % step < 0) + 1);
    return k <= hi && from + k * step < a_width;
}

constexpr int64_t kMostSteps = 1 << 22;

inline bool meet(const Runs& a, const Runs& b) {
    if (a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0 || a.at >= b.at + b.span() || b.at >= a.at + a.span()) return false;
    int64_t left = kMostSteps;
    auto rows_meet = [&](int64_t from) {
        if (a.rows == 1 || b.rows == 1 || a.row == b.row)       // (one step counts, or the rows' difference)
            return steps_meet(from, b.rows == 1 ? a.row : b.row, 1 - a.rows, b.rows - 1, a.width, b.width);
        const int64_t all = std::gcd(a.row, b.row);
        if (!steps_meet(from, all, -(1ll << 40), 1ll << 40, a.width, b.width)) return false;
        for (int64_t i = 0; i < a.rows; ++i)
            if (--left < 0 || steps_meet(from - i * a.row, b.row, 0, b.rows - 1, a.width, b.width)) return true;
        return false;
    };
    const int64_t from = b.at - a.at;
    if (a.heads == 1 || b.heads == 1 || a.head == b.head) {     // heads that lie equally far apart: their difference counts
        const int64_t head = b.heads == 1 ? a.head : b.head;
        for (int64_t m = 1 - a.heads; m < b.heads; ++m)
            if (--left < 0 || rows_meet(from + m * head)) return true;
        return false;
    }
    for (int64_t i = 0; i < a.heads; ++i)
        for (int64_t j = 0; j < b.heads; ++j)
            if (--left < 0 || rows_meet(from + j * b.head - i * a.head)) return true;
    return false;
}

}  // namespace tsp
