// Small random regions against their bytes: overlap() never claims what is not
// so, and misses nothing where it says that it is exact.
#include <cstdio>
#include <random>
#include <set>

#include "overlap.hpp"

using vkfx::Region;

static std::set<uintptr_t> bytes(const Region& r) {
    std::set<uintptr_t> s;
    for (uint64_t i = 0; i < r.extent[0]; ++i)
        for (uint64_t j = 0; j < r.extent[1]; ++j)
            for (uint64_t k = 0; k < r.extent[2]; ++k)
                for (uint64_t e = 0; e < r.run; ++e) s.insert(r.at + i * r.stride[0] + j * r.stride[1] + k * r.stride[2] + e);
    return s;
}

// no axis' runs reach past the next of a larger one
static bool nested(const Region& r) {
    vkfx::overlap_detail::Axis axes[3];
    uint64_t span = r.run;
    for (int n = vkfx::overlap_detail::sorted(r, axes); n--; span += axes[n].stride * (uint64_t)axes[n].high)
        if (axes[n].stride < span) return false;
    return true;
}

int main() {
    std::mt19937 rng(7);
    const auto pick = [&](int lo, int hi) { return (uint64_t)std::uniform_int_distribution<int>(lo, hi)(rng); };
    long claims = 0, exact = 0, all = 0;
    for (int round = 0; round < 200000; ++round) {
        Region a, b;
        a.at = 1000 + pick(0, 40), b.at = 1000 + pick(0, 40);
        a.run = pick(0, 6), b.run = pick(0, 6);
        const bool same = pick(0, 1);
        uint64_t order[3] = {0, 1, 2};
        std::shuffle(order, order + 3, rng);
        uint64_t sa = a.run, sb = b.run;
        for (int i = 0; i < 3; ++i) {  // mostly nested
            const uint64_t s = pick(0, 9) ? std::max(sa, same ? sb : sa) + pick(0, 5) : pick(0, 12);
            const uint64_t t = same ? s : (pick(0, 9) ? sb + pick(0, 5) : pick(0, 12)), na = pick(1, 4), nb = pick(1, 4);
            a.axis((int)order[i], s, na), b.axis((int)order[i], t, nb);
            sa += s * (na - 1), sb += t * (nb - 1);
        }
        const std::set<uintptr_t> x = bytes(a), y = bytes(b);
        bool want = false;
        for (uintptr_t p : x) want = want || y.count(p);
        const bool got = vkfx::overlap(a, b), turned = vkfx::overlap(b, a);
        if ((got || turned) && !want) return printf("claims an overlap that is none in round %d\n", round), 1;
        ++all;
        claims += got;
        using vkfx::overlap_detail::dense;
        Region both;  // what holds the two if their strides are the same
        both.run = std::max(a.run, b.run);
        for (int i = 0; i < 3; ++i)
            both.axis(i, a.extent[i] > 1 ? a.stride[i] : b.stride[i], std::max(a.extent[i], b.extent[i]));
        if ((same && nested(both)) || (dense(a) && nested(b)) || (dense(b) && nested(a))) {
            ++exact;
            if (got != want || turned != want) return printf("misses an overlap in round %d\n", round), 1;
        }
    }
    if (exact < all / 4 || claims < all / 10) return printf("too few cases: %ld exact, %ld overlaps\n", exact, claims), 1;
    // offsets past 32 bits
    Region p, q;
    p.at = 1 << 20, q.at = (1 << 20) + 256;
    p.run = q.run = 256;
    p.axis(0, 1ull << 40, 5).axis(1, 1ull << 20, 9), q.axis(0, 1ull << 40, 5).axis(1, 1ull << 20, 9);
    if (vkfx::overlap(p, q)) return printf("interleaved rows\n"), 1;
    q.at += (3ull << 40) + (7ull << 20) - 1;
    if (!vkfx::overlap(p, q)) return printf("far rows\n"), 1;
    printf("ok %ld cases, %ld exact, %ld overlaps\n", all, exact, claims);
    return 0;
}
