// Whether a call's arrays overlap, by their addresses.  Plain C++, so that a host test can
// compile it.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace pk {

inline bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    return a && b && (const char*)a < (const char*)b + b_bytes && (const char*)b < (const char*)a + a_bytes;
}

// Rows of `width` bytes, `stride` >= width apart.
struct RowSet {
    const void* base;
    int64_t stride, width, rows;
    int64_t extent() const { return (rows - 1) * stride + width; }
};
inline bool overlap(const RowSet& r, const void* p, int64_t bytes) {
    if (!p || bytes <= 0 || r.rows <= 0) return false;
    const int64_t d = (const char*)p - (const char*)r.base;  // in question: the first row that ends behind p
    const int64_t first = d < r.width ? 0 : (d - r.width) / r.stride + 1;
    return first < r.rows && first * r.stride < d + bytes;
}
// Slices of one array's rows lie between each other without meeting: in question are single rows.
inline bool overlap(const RowSet& a, const RowSet& b) {
    if (a.rows <= 0 || b.rows <= 0 || !overlap(a.base, a.extent(), b.base, b.extent())) return false;
    if (a.stride == b.stride) {  // rows i of a and j of b meet or not by i - j: in question is the first that ends behind b's
        const int64_t s = a.stride, d = (const char*)b.base - (const char*)a.base, e = d - a.width;
        const int64_t above = (e >= 0 ? e / s : -((-e + s - 1) / s)) + 1, first = above > 1 - b.rows ? above : 1 - b.rows;
        return first < a.rows && first * s < d + b.width;
    }
    for (int64_t i = 0; i < b.rows; ++i)
        if (overlap(a, (const char*)b.base + i * b.stride, b.width)) return true;
    return false;
}

}  // namespace pk
