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

}  // namespace plan
}  // namespace fgqa
