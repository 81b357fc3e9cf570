// row_span.hpp -- do two strided sets of rows share memory?  Host side; what the operators' argument checks ask (linear_ops.cpp).
#pragma once

#include <algorithm>
#include <cstdint>

namespace mi355 {

// Rows of `row_bytes` bytes, repeated over up to two axes (rows of a matrix, entries of a batch; in memory order, so [batch][rows] and
// [rows][batch] are the same set): the longer step first, an axis of one entry or none to step over is {1, 0}.
struct row_span {
    struct axis { uint64_t count, step; };
    uintptr_t at;             // first byte
    uint64_t row_bytes;       // 0: nothing
    axis axes[2];
    uintptr_t end() const { return at + (axes[0].count - 1) * axes[0].step + (axes[1].count - 1) * axes[1].step + row_bytes; }
};

constexpr row_span NO_SPAN{0, 0, {{1, 0}, {1, 0}}};

inline row_span span_of(const void *p, int64_t rows, int64_t cols, int64_t ld, int64_t esz, int64_t batch = 1, int64_t stride = 0)
{
    if (!p || rows <= 0 || cols <= 0 || batch <= 0) return NO_SPAN;
    auto axis = [&](int64_t count, int64_t step) { return count == 1 || step == 0 ? row_span::axis{1, 0} : row_span::axis{(uint64_t)count, (uint64_t)(step * esz)}; };
    row_span s{reinterpret_cast<uintptr_t>(p), (uint64_t)(cols * esz), {axis(rows, ld), axis(batch, stride)}};
    if (s.axes[0].step < s.axes[1].step) std::swap(s.axes[0], s.axes[1]);
    const uint64_t c0 = s.axes[0].count, c1 = s.axes[1].count, s0 = s.axes[0].step, s1 = s.axes[1].step;
    if (c1 > 1 && s0 == c1 * s1) s.axes[0] = {c0 * c1, s1}, s.axes[1] = {1, 0};      // one follows on from the other
    else if (c1 > 1 && s0 == s1) s.axes[0].count = c0 + c1 - 1, s.axes[1] = {1, 0};  // or both step the same way
    return s;
}

enum { SPANS_APART = 0, SPANS_SAME = 1, SPANS_OVERLAP = 2 };

// Exact where the two sets step by the same (at most two) distances, as parts of one larger tensor do; sets that step differently and whose
// extents meet are taken as sharing memory.
inline int spans_relation(const row_span &a, const row_span &b)
{
    if (!a.row_bytes || !b.row_bytes || a.end() <= b.at || b.end() <= a.at) return SPANS_APART;
    auto same = [](const row_span::axis &x, const row_span::axis &y) { return x.count == y.count && x.step == y.step; };
    if (a.at == b.at && a.row_bytes == b.row_bytes && same(a.axes[0], b.axes[0]) && same(a.axes[1], b.axes[1])) return SPANS_SAME;
    // the distances, and how often each set takes each of them
    struct { int64_t step = 0, na = 1, nb = 1; } dim[2];
    int dims = 0;
    for (int side = 0; side < 2; ++side)
        for (const row_span::axis &x : side ? b.axes : a.axes) {
            if (x.count == 1) continue;
            int d = 0;
            while (d < dims && dim[d].step != (int64_t)x.step) ++d;
            if (d == 2) return SPANS_OVERLAP;
            if (d == dims) dim[dims++].step = (int64_t)x.step;
            (side ? dim[d].nb : dim[d].na) = (int64_t)x.count;
        }
    // Rows i and j of the two overlap where b's begins less than a row before or behind a's: -row_b < distance + i step0 + j step1 < row_a, with
    // i and j differences of row numbers.  One of them is walked, the other solved for.
    if (dim[0].na + dim[0].nb < dim[1].na + dim[1].nb) std::swap(dim[0], dim[1]);
    if (dim[1].na + dim[1].nb > 1 << 18) return SPANS_OVERLAP;
    const int64_t wa = (int64_t)a.row_bytes, wb = (int64_t)b.row_bytes, distance = (int64_t)(b.at - a.at);
    auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0 ? 1 : 0); };
    for (int64_t j = 1 - dim[1].na; j < dim[1].nb; ++j) {
        const int64_t x = distance + j * dim[1].step;
        if (dim[0].step == 0) {
            if (-wb < x && x < wa) return SPANS_OVERLAP;
            continue;
        }
        const int64_t first = std::max(floor_div(-wb - x, dim[0].step) + 1, 1 - dim[0].na), last = std::min(floor_div(wa - 1 - x, dim[0].step), dim[0].nb - 1);
        if (first <= last) return SPANS_OVERLAP;
    }
    return SPANS_APART;
}

// Does entry b of a batch begin where no other entry lies?  One behind the other, or their rows in turn.
inline bool entries_apart(int64_t batch, int64_t rows, int64_t cols, int64_t ld, int64_t stride)
{
    return batch <= 1 || stride >= (rows - 1) * ld + cols || (stride >= cols && ld >= (batch - 1) * stride + cols);
}

}  // namespace mi355
