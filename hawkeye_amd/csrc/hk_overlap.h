// Host-side checks of what a call writes: that its rows are apart, and apart from what it reads.
#pragma once
#include <stdint.h>

// Host-side check that what a call writes shares no byte with what it reads: an operand of n1 x n2 rows of `row` elements (strides in
// elements, not negative), from its first byte a to the one behind its last, b.  A null operand has no rows.
struct HkSpan {
    uintptr_t a, b;
    int64_t n1, s1, n2, s2, row;     // in bytes
};
static inline HkSpan hk_span(const void* ptr, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t row, int64_t elem) {
    if (!ptr || n1 < 1 || n2 < 1 || row < 1) return {};
    const uintptr_t a = reinterpret_cast<uintptr_t>(ptr);
    return {a, a + (uintptr_t)(((n1 - 1) * s1 + (n2 - 1) * s2 + row) * elem), n1, s1 * elem, n2, s2 * elem, row * elem};
}
// Pieces of x and y that begin at a + (whole multiples of g) and are px and py bytes long never meet if they lie side by side within g.
static inline bool hk_side_by_side(uintptr_t xa, int64_t px, uintptr_t ya, int64_t py, uint64_t g) {
    if (g == 0) return false;
    const uint64_t d = ya >= xa ? (ya - xa) % g : (g - (xa - ya) % g) % g;      // y's place within x's period
    return d >= (uint64_t)px && d + (uint64_t)py <= g;
}
// Operands interleaved in one tensor (K and V of a cache [B, rows, 2, H, hd] or [B, 2, rows, H, hd]) do not overlap, though their spans do: rows,
// or the whole blocks that one index leaves, lie side by side.  May find an overlap where a layout is more intricate than that, never the reverse.
static inline bool hk_overlap(const HkSpan& x, const HkSpan& y) {
    if (x.a >= y.b || y.a >= x.b) return false;
    auto gcd = [](int64_t p, int64_t q) {
        while (q) {
            const int64_t r = p % q;
            p = q;
            q = r;
        }
        return p;
    };
    const int64_t g1 = gcd(x.n1 > 1 ? x.s1 : 0, y.n1 > 1 ? y.s1 : 0), g2 = gcd(x.n2 > 1 ? x.s2 : 0, y.n2 > 1 ? y.s2 : 0);
    return !hk_side_by_side(x.a, x.row, y.a, y.row, gcd(g1, g2)) &&
           !hk_side_by_side(x.a, (x.n2 - 1) * x.s2 + x.row, y.a, (y.n2 - 1) * y.s2 + y.row, g1) &&
           !hk_side_by_side(x.a, (x.n1 - 1) * x.s1 + x.row, y.a, (y.n1 - 1) * y.s1 + y.row, g2);
}

// Rows of `row` elements at i1 * s1 + i2 * s2 (i1 < n1, i2 < n2) that a call writes: no two share an element, the one index within the other's steps.
static inline bool hk_rows_apart(int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t row) {
    if ((n1 > 1 && s1 < row) || (n2 > 1 && s2 < row)) return false;
    return n1 <= 1 || n2 <= 1 || s1 >= (n2 - 1) * s2 + row || s2 >= (n1 - 1) * s1 + row;
}
