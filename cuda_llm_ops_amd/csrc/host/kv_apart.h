// Whether two views of the same kind share memory (host only).
#pragma once

#include <stdint.h>

namespace fgqa {
namespace plan {

// Whether an element of the view at byte `a` and one of the view at byte `b` meet:
// both of n[i] elements, `elem` bytes each, at strides s[i] (in elements) in k dims,
// whose own elements lie apart.  Exact where the strides nest (each at least the span
// of the smaller ones), as those of such a view do; dims of one element do not count.
inline bool views_meet(uintptr_t a, uintptr_t b, const int64_t* n, const int64_t* s, int k, int64_t elem) {
    typedef __int128 i128;
    constexpr int kMost = 8;
    i128 step[kMost], count[kMost], span[kMost];   // by falling stride; span: bytes from the first to past the last
    int dims = 0;
    for (int i = 0; i < k; ++i) {
        if (n[i] <= 0) return false;
        if (n[i] == 1) continue;
        if (dims == kMost) return true;   // (never: views of at most 4 dims)
        int at = dims++;
        for (; at > 0 && step[at - 1] < (i128)s[i] * elem; --at) {
            step[at] = step[at - 1];
            count[at] = count[at - 1];
        }
        step[at] = (i128)s[i] * elem;
        count[at] = n[i];
    }
    i128 inner = elem;
    for (int i = dims - 1; i >= 0; --i) inner = span[i] = inner + (count[i] - 1) * step[i];
    // b - a as sum of x[i] * step[i] with |x[i]| < count[i], less than an element
    // off: x[i] is the quotient rounded down, or one more
    struct Search {
        const i128 *step, *count, *span;
        int dims;
        i128 elem;
        bool at(int i, i128 d) const {
            if (i == dims) return d < elem && d > -elem;
            if (d >= span[i] || d <= -span[i]) return false;
            if (step[i] == 0) return true;   // (elements of one view meet)
            i128 x = d / step[i];
            if (d < 0 && x * step[i] != d) --x;
            for (int e = 0; e < 2; ++e, ++x)
                if (x < count[i] && -x < count[i] && at(i + 1, d - x * step[i])) return true;
            return false;
        }
    };
    return Search{step, count, span, dims, elem}.at(0, (i128)b - (i128)a);
}

// Blocks of len_a bytes at a + i s0 + j s1 and of len_b bytes at b + i s0 + j s1, for every
// i < n0 and j < n1 (strides in bytes, 0 or more): whether one of the first meets one of
// the second.  Exact where the strides nest; true for some that do not.
inline bool blocks_meet(uintptr_t a, int64_t len_a, uintptr_t b, int64_t len_b, int64_t n0, int64_t s0, int64_t n1, int64_t s1) {
    if (n0 <= 0 || n1 <= 0 || len_a <= 0 || len_b <= 0) return false;
    typedef __int128 i128;
    // b - a = x s0 + y s1 + d with |x| < n0, |y| < n1 and -len_b < d < len_a; the larger
    // stride first
    if (s0 < s1) {
        int64_t t = s0;
        s0 = s1;
        s1 = t;
        t = n0;
        n0 = n1;
        n1 = t;
    }
    auto floor_div = [](i128 x, i128 y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
    auto inner = [&](i128 d) {   // some |y| < n1 with -len_b < d - y s1 < len_a
        if (s1 == 0 || n1 == 1) return d < len_a && d > -(i128)len_b;
        // y from the least with d - y s1 < len_a
        i128 y = floor_div(d - len_a, s1) + 1;
        if (y < -(i128)(n1 - 1)) y = -(i128)(n1 - 1);
        return y < n1 && d - y * s1 > -(i128)len_b && d - y * s1 < len_a;
    };
    const i128 d = (i128)b - (i128)a;
    if (s0 == 0 || n0 == 1) return inner(d);
    // what the inner blocks span on either side
    const i128 reach = (i128)(n1 - 1) * s1 + (len_a > len_b ? len_a : len_b);
    i128 lo = floor_div(d - reach, s0), hi = floor_div(d + reach, s0) + 1;
    if (lo < -(i128)(n0 - 1)) lo = -(i128)(n0 - 1);
    if (hi > n0 - 1) hi = n0 - 1;
    if (hi - lo > 64) return true;   // (strides that do not nest)
    for (i128 x = lo; x <= hi; ++x)
        if (inner(d - x * s0)) return true;
    return false;
}

}  // namespace plan
}  // namespace fgqa
