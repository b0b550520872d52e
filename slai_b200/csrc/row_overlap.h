// Whether two sets of rows in device memory share a float.  Plain C++ (the tests compile it by itself).
#pragma once
#include <stdint.h>

// n rows each, of `w` floats, `ld` >= w floats apart; a and b are the addresses of the first ones.  Exact: rows of one product's parts lie between one another.
inline bool rows_overlap(uintptr_t a, int64_t ld_a, int64_t w_a, uintptr_t b, int64_t ld_b, int64_t w_b, int64_t n) {
    typedef __int128 wide;
    if (n <= 0 || w_a <= 0 || w_b <= 0) return false;
    const wide A = a, B = b, la = (wide)4 * ld_a, lb = (wide)4 * ld_b, wa = (wide)4 * w_a, wb = (wide)4 * w_b;
    if (B >= A + (n - 1) * la + wa || A >= B + (n - 1) * lb + wb) return false;  // one behind the other
    if (n == 1) return true;
    if (la == lb) {  // row j of b begins d bytes behind row j + k of a
        const wide by = B - A;
        wide k, d;
        if (la < (wide)1 << 62 && by < (wide)1 << 62 && -by < (wide)1 << 62) {  // (the wide division takes longer)
            const int64_t L = (int64_t)la, x = (int64_t)by, q = x / L;
            k = q - (x - q * L < 0);
            d = by - k * la;
        } else {
            k = by / la - (by % la < 0);
            d = by - k * la;
        }
        auto there = [&](wide rows) { return rows < n && -rows < n; };
        return (d < wa && there(k)) || (d + wb > la && there(k + 1));
    }
    for (int64_t i = 0, j = 0; i < n && j < n;) {
        const wide x = A + i * la, y = B + j * lb;
        if (x + wa <= y) i++;
        else if (y + wb <= x) j++;
        else return true;
    }
    return false;
}
