// overlap.cuh -- whether rows of memory share bytes, from their addresses, extents and
// strides alone (host).
#pragma once

#include <stdint.h>

namespace spark {

// Rows of n values of `item` bytes: a row for each place of up to three dimensions, their strides in values (one of extent 1
// has none).
struct Rows {
    const void* at;
    int64_t item, n;
    int dims;
    int64_t extent[3], stride[3];
};

namespace overlap {
using Wide = __int128;
// A step that is taken lo to hi times.
struct Step {
    Wide step, lo, hi;
};
// What steps, the longest first, and lo to hi bytes come to.
struct Sum {
    Step steps[6];
    int n = 0;
    Wide lo = 0, hi = 0;
    void add(Wide step, Wide lo, Wide hi) {
        int i = 0;
        while (i < n && steps[i].step > step) ++i;
        if (i < n && steps[i].step == step) {
            steps[i].lo += lo, steps[i].hi += hi;
            return;
        }
        for (int k = n++; k > i; --k) steps[k] = steps[k - 1];
        steps[i] = Step{step, lo, hi};
    }
    // Whether the steps from the i-th on and the bytes may come to d; `left` is how often that may be asked.
    bool reaches(Wide d, int i, int& left) const {
        if (--left < 0) return false;
        if (i == n) return lo <= d && d <= hi;
        Wide low = lo, high = hi;
        for (int k = i + 1; k < n; ++k) low += steps[k].step * steps[k].lo, high += steps[k].step * steps[k].hi;
        const Step& s = steps[i];
        Wide from = down(d - high + s.step - 1, s.step), to = down(d - low, s.step);
        if (from < s.lo) from = s.lo;
        if (to > s.hi) to = s.hi;
        for (Wide k = from; k <= to && left > 0; ++k)
            if (reaches(d - k * s.step, i + 1, left)) return true;
        return false;
    }
    static Wide down(Wide a, Wide b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }
};
// The rows' first byte, and their steps (all above 0).
inline Wide first(const Rows& r, Sum& sum, bool back) {
    Wide at = (Wide)reinterpret_cast<uintptr_t>(r.at);
    for (int i = 0; i < r.dims; ++i) {
        const Wide step = (Wide)r.stride[i] * r.item, last = r.extent[i] - 1;
        if (last <= 0 || step == 0) continue;
        if (step < 0) at += last * step;
        sum.add(step < 0 ? -step : step, back ? -last : 0, back ? 0 : last);
    }
    const Wide bytes = (Wide)r.n * r.item - 1;
    (back ? sum.lo : sum.hi) = back ? -bytes : bytes;
    return at;
}
// The rows' bytes from the first to behind the last; whole numbers below 2^53.
inline void range(const Rows& r, double& from, double& to) {
    from = (double)reinterpret_cast<uintptr_t>(r.at), to = from + (double)r.n * (double)r.item;
    for (int i = 0; i < r.dims; ++i) {
        const double all = (double)(r.extent[i] - 1) * (double)r.stride[i] * (double)r.item;
        (all < 0 ? from : to) += all;
    }
}
inline bool empty(const Rows& r) {
    bool none = r.n <= 0;
    for (int i = 0; i < r.dims; ++i) none = none || r.extent[i] <= 0;
    return none;
}
}  // namespace overlap

// Whether each row has bytes of its own.  (By dimensions that lie in one another, a longer stride behind all rows of the shorter
// ones: rows that are apart in another way count as not.)
inline bool rows_apart(const Rows& r) {
    if (overlap::empty(r)) return true;
    overlap::Sum sum;
    overlap::first(r, sum, false);
    int dims = 0;
    for (int i = 0; i < r.dims; ++i) dims += r.extent[i] > 1;
    overlap::Wide bytes = sum.hi + 1;
    if (sum.n < dims) return false;      // (equal strides, or a stride of 0)
    for (int i = sum.n - 1; i >= 0; --i) {
        if (sum.steps[i].step < bytes) return false;
        bytes += sum.steps[i].step * sum.steps[i].hi;
    }
    return true;
}

// Whether a row of a shares bytes with one of b: whether b's address less a's is a sum of their strides, each an allowed number of times,
// and of places in a row.  Strides of one order, as two parts of a tensor have them, leave two numbers to try for each; where
// others leave too many, it is not said.
inline bool rows_meet(const Rows& a, const Rows& b) {
    if (overlap::empty(a) || overlap::empty(b)) return false;
    double a0, a1, b0, b1;
    overlap::range(a, a0, a1), overlap::range(b, b0, b1);
    if ((a1 <= b0 || b1 <= a0) && a0 > -0x1p52 && b0 > -0x1p52 && a1 < 0x1p52 && b1 < 0x1p52) return false;
    overlap::Sum sum;
    const overlap::Wide from = overlap::first(a, sum, false), to = overlap::first(b, sum, true);
    int left = 1 << 12;
    return sum.reaches(to - from, 0, left);
}

}  // namespace spark
