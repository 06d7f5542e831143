// row_overlap.h — whether two sets of equally spaced rows share memory (no HIP in here: it builds with a plain C++ compiler).
#pragma once
#include <stdint.h>

namespace oxb {

// `n` rows of `wide` bytes, `stride` (>= wide) bytes apart; n and wide at least 1.
struct RowSpan {
    uint64_t at, n, wide, stride;
};

// Rows side by side in one wider buffer (the q heads and the outputs of a product's rows) do not overlap, though their ranges do.
inline bool rows_overlap(const RowSpan& a, const RowSpan& b) {
    typedef __int128 wide_t;  // (rows times stride may pass 64 bits)
    auto end = [](const RowSpan& s) { return (wide_t)s.at + (wide_t)(s.n - 1) * s.stride + s.wide; };
    if (end(a) <= (wide_t)b.at || end(b) <= (wide_t)a.at) return false;
    if (a.n == 1 || b.n == 1 || a.stride != b.stride) {
        // the two in order of addresses, each time on to the first row that ends behind the other's begin
        uint64_t i = 0, j = 0;
        while (i < a.n && j < b.n) {
            const wide_t x = (wide_t)a.at + (wide_t)i * a.stride, y = (wide_t)b.at + (wide_t)j * b.stride;
            if (x + a.wide <= y) i += (uint64_t)((y - x - a.wide) / a.stride) + 1;
            else if (y + b.wide <= x) j += (uint64_t)((x - y - b.wide) / b.stride) + 1;
            else return true;
        }
        return false;
    }
    // row j of b lies d + (j - i) stride behind row i of a: they overlap where that is above -b.wide and below a.wide
    const wide_t d = (wide_t)b.at - (wide_t)a.at, s = a.stride, low = -(wide_t)b.wide - d;
    wide_t k = low >= 0 ? low / s + 1 : -((-low + s - 1) / s) + 1;  // the smallest k with d + k s > -b.wide
    if (k < -(wide_t)(a.n - 1)) k = -(wide_t)(a.n - 1);
    return k <= (wide_t)(b.n - 1) && d + k * s < (wide_t)a.wide;
}

}  // namespace oxb
