// Do the address ranges of the matrices of a clipping call lie apart?  Six
// integers per matrix: A, lda, B, ldb, rows, columns; ea and eb bytes per
// element.  A matrix that is scaled in place (same memory, same type) counts once.
#pragma once
#include <algorithm>
#include <cstdint>
#include <vector>

inline bool clip_apart(const int64_t* v, size_t count, int ea, int eb) {
    std::vector<int64_t> lo, hi;
    lo.reserve(2 * count);
    hi.reserve(2 * count);
    auto add = [&](int64_t p, int64_t ld, int64_t rows, int64_t cols, int es) {
        lo.push_back(p);
        hi.push_back(p + ((cols - 1) * ld + rows) * es);
    };
    for (size_t i = 0; i < count; ++i, v += 6) {
        if (v[4] <= 0 || v[5] <= 0) continue;
        add(v[2], v[3], v[4], v[5], eb);
        if (v[0] != v[2] || v[1] != v[3] || ea != eb) add(v[0], v[1], v[4], v[5], ea);
    }
    // disjoint intervals: each ends before the next begins
    std::sort(lo.begin(), lo.end());
    std::sort(hi.begin(), hi.end());
    for (size_t i = 1; i < lo.size(); ++i)
        if (hi[i - 1] > lo[i]) return false;
    return true;
}
