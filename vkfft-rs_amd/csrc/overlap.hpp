// overlap.hpp -- whether two strided tensors share memory, as far as it can be
// told without going through their elements.
#pragma once

#include <algorithm>
#include <cstdint>

namespace vkfx {

// Runs of `run` bytes at `at` + a multiple of each axis' stride, in bytes.
struct Region {
    uintptr_t at = 0;
    uint64_t run = 0;  // 0: nothing
    uint64_t stride[3] = {0, 0, 0};
    uint64_t extent[3] = {1, 1, 1};

    // An axis of `n` places `s` bytes apart; a broadcast one adds none.
    Region& axis(int i, uint64_t s, uint64_t n) {
        if (!n) run = 0;
        stride[i] = s;
        extent[i] = s && n > 1 ? n : 1;
        return *this;
    }
    uint64_t span() const {
        uint64_t n = run;
        for (int i = 0; i < 3; ++i) n += stride[i] * (extent[i] - 1);
        return n;
    }
};

namespace overlap_detail {

struct Axis {
    uint64_t stride;
    int64_t low, high;  // of the difference of two tensors' places
};

// Axes by their strides, the largest first; without those of one place.
inline int sorted(const Region& r, Axis (&axes)[3]) {
    int n = 0;
    for (int i = 0; i < 3; ++i)
        if (r.extent[i] > 1) axes[n++] = Axis{r.stride[i], 0, (int64_t)r.extent[i] - 1};
    std::sort(axes, axes + n, [](const Axis& x, const Axis& y) { return x.stride > y.stride; });
    return n;
}

// Whether some places have a run of `a` and one of `b` meet that start `apart` bytes (b - a) from each other.
inline bool reaches(const Axis* axes, int n, int64_t apart, int64_t a, int64_t b) {
    if (!n) return apart < a && -apart < b;
    const int64_t s = (int64_t)axes->stride;
    const int64_t floor = apart >= 0 ? apart / s : -((-apart + s - 1) / s);
    for (int64_t d = floor; d <= floor + 1; ++d)
        if (d >= axes->low && d <= axes->high && reaches(axes + 1, n - 1, apart - d * s, a, b)) return true;
    return false;
}

inline bool dense(const Region& r) {
    Axis axes[3];
    uint64_t span = r.run;
    for (int n = sorted(r, axes); n--; span += axes[n].stride * (uint64_t)axes[n].high)
        if (axes[n].stride > span) return false;
    return true;
}

// Whether runs of `r` meet the bytes [low, high).
inline bool meets(const Region& r, uintptr_t low, uintptr_t high) {
    if (high <= r.at) return false;
    // the last run that starts before `high`, as far as axes do not interleave
    Axis axes[3];
    const int n = sorted(r, axes);
    uint64_t left = high - 1 - r.at;
    uintptr_t start = r.at;
    for (int i = 0; i < n; ++i) {
        const uint64_t k = std::min((uint64_t)axes[i].high, left / axes[i].stride);
        start += k * axes[i].stride;
        left -= k * axes[i].stride;
    }
    return start + r.run > low;
}

}  // namespace overlap_detail

// True only where the two do share memory. Told exactly where one of them has
// no gaps, or where both have the strides of one layout, in which no axis' runs
// reach past the next of a larger one; otherwise false may be wrong.
inline bool overlap(const Region& a, const Region& b) {
    using namespace overlap_detail;
    if (!a.run || !b.run || a.at >= b.at + b.span() || b.at >= a.at + a.span()) return false;
    if (dense(a)) return meets(b, a.at, a.at + a.span());
    if (dense(b)) return meets(a, b.at, b.at + b.span());
    Axis axes[3];
    int n = 0;
    for (int i = 0; i < 3; ++i) {
        if (a.extent[i] == 1 && b.extent[i] == 1) continue;
        if (a.extent[i] > 1 && b.extent[i] > 1 && a.stride[i] != b.stride[i]) return false;
        axes[n++] = Axis{a.extent[i] > 1 ? a.stride[i] : b.stride[i], 1 - (int64_t)b.extent[i], (int64_t)a.extent[i] - 1};
    }
    std::sort(axes, axes + n, [](const Axis& x, const Axis& y) { return x.stride > y.stride; });
    return reaches(axes, n, (int64_t)(b.at - a.at), (int64_t)a.run, (int64_t)b.run);
}

}  // namespace vkfx
