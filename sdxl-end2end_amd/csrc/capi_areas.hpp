// Which bytes the tensors of a C ABI call occupy, and whether two of them share any.
#pragma once

#include <cstdint>
#include <initializer_list>

namespace sdxl_hip {

// What a tensor occupies: rows of `row` bytes, `stride` bytes apart.
struct Area {
    const void* p;
    int64_t rows, row, stride;
};

inline Area matrix(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t elem = 2) {
    return {p, rows, cols * elem, ld * elem};
}
inline Area vector(const void* p, int64_t n, int64_t elem = 2) { return {p, 1, n * elem, n * elem}; }

using i128 = __int128;  // (offsets of two 63-bit areas)

inline i128 floor_div(i128 a, i128 b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }

// Whether two areas share a byte. Slices of one wide tensor lie between each other's rows and share none: seen where
// the strides are equal or one of the areas is a single run of bytes. Of others, which lie between each other with
// different strides, only the first and last rows are looked at.
inline bool overlap(Area a, Area b) {
    if (a.p == nullptr || b.p == nullptr || a.rows <= 0 || b.rows <= 0 || a.row <= 0 || b.row <= 0) return false;
    const i128 d = (i128)(uintptr_t)b.p - (i128)(uintptr_t)a.p;  // b's begin from a's
    for (Area* t : {&a, &b})
        if (t->rows == 1 || t->stride == t->row) *t = {t->p, 1, t->rows * t->row, 0};
    if (a.rows > 1 && b.rows > 1 && a.stride != b.stride) {
        const auto row = [](const Area& t, int64_t r) { return Area{(const char*)t.p + r * t.stride, 1, t.row, 0}; };
        return overlap(row(a, 0), b) || overlap(row(a, a.rows - 1), b) || overlap(row(b, 0), a) || overlap(row(b, b.rows - 1), a);
    }
    if (a.rows == 1 && b.rows == 1) return d - a.row < 0 && d + b.row > 0;
    // a's row i meets b's row j where (i - j) stride lies in (d - a.row, d + b.row): the least such i - j
    const i128 stride = a.rows > 1 ? a.stride : b.stride;
    i128 t = floor_div(d - a.row, stride) + 1;
    if (t < -(i128)(b.rows - 1)) t = -(i128)(b.rows - 1);
    return t <= a.rows - 1 && t * stride < d + b.row;
}

inline bool overlaps_one(Area out, std::initializer_list<Area> inputs) {
    for (const Area& in : inputs)
        if (overlap(out, in)) return true;
    return false;
}

}  // namespace sdxl_hip
