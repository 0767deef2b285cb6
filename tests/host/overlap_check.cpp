// Random layouts of heads, byte by byte against tsp::meet: views that interleave, lie on each other at an offset, are dense, have
// broadcast strides or strides of their own. Host code alone.
#include <cstdio>
#include <random>
#include <vector>

#include "overlap.hpp"

static bool share_a_byte(const tsp_heads& a, int64_t na, int ha, int da, const tsp_heads& b, int64_t nb, int hb, int db, size_t size) {
    std::vector<char> held(1 << 16, 0);
    auto each = [&](const tsp_heads& t, int64_t n, int heads, int d, auto f) {
        for (int64_t i = 0; i < n; ++i)
            for (int h = 0; h < heads; ++h)
                for (int64_t e = 0; e < d * (int64_t)size; ++e)
                    f((int64_t)reinterpret_cast<uintptr_t>(t.data) + (i * t.row_stride + h * t.head_stride) * (int64_t)size + e);
    };
    bool any = false;
    each(a, na, ha, da, [&](int64_t at) { held.at(at) = 1; });
    each(b, nb, hb, db, [&](int64_t at) { any |= held.at(at) != 0; });
    return any;
}

int main() {
    std::mt19937 rng(1);
    auto pick = [&](std::initializer_list<int> v) { return v.begin()[rng() % v.size()]; };
    int met = 0, apart = 0, interleaved = 0;
    for (int i = 0; i < 300000; ++i) {
        const size_t size = pick({2, 4});
        const int da = pick({8, 16, 24}), db = rng() % 4 ? da : pick({8, 16, 24}), ha = pick({1, 1, 2, 3, 4}), hb = rng() % 2 ? ha : pick({1, 2, 3, 5});
        const int64_t na = pick({1, 2, 3, 7}), nb = rng() % 2 ? na : pick({1, 2, 4, 9});
        auto at = [&] { return reinterpret_cast<void*>((uintptr_t)(64 + 16 * (rng() % 80))); };
        tsp_heads a{at(), 8 * (int64_t)(rng() % 24), 8 * (int64_t)(rng() % 12)}, b{at(), rng() % 2 ? a.row_stride : 8 * (int64_t)(rng() % 24),
                                                                                 rng() % 2 ? a.head_stride : 8 * (int64_t)(rng() % 12)};
        if (rng() % 16 == 0) b.head_stride = na * a.row_stride;      // heads outside the rows
        const tsp::Runs ra = tsp::runs_of(a, na, ha, da, size), rb = tsp::runs_of(b, nb, hb, db, size);
        const bool want = share_a_byte(a, na, ha, da, b, nb, hb, db, size), spans = ra.at < rb.at + rb.span() && rb.at < ra.at + ra.span();
        if (tsp::meet(ra, rb) != want || tsp::meet(rb, ra) != want) {
            std::printf("case %d: %d expected\n", i, want);
            return 1;
        }
        if (want) ++met;
        else if (spans) ++interleaved;
        else ++apart;
    }
    // far strides and many rows, which take no steps a row
    const tsp_heads q{reinterpret_cast<void*>(uintptr_t{1} << 40), 1 << 20, 128}, k{reinterpret_cast<void*>((uintptr_t{1} << 40) + 4096), 1 << 20, 128};
    const int64_t n = (1ll << 31) - 1;
    if (tsp::meet(tsp::runs_of(q, n, 16, 128, 2), tsp::runs_of(k, n, 16, 128, 2)) || !tsp::meet(tsp::runs_of(q, n, 17, 128, 2), tsp::runs_of(k, n, 16, 128, 2))) return 2;
    // nothing, and one run
    if (tsp::meet(tsp::runs_of(nullptr, 100), tsp::runs_of(q, n, 16, 128, 2)) || tsp::meet(tsp::runs_of(q.data, 0), tsp::runs_of(q, n, 16, 128, 2))) return 3;
    if (!tsp::meet(tsp::runs_of(q.data, 1), tsp::runs_of(q, n, 16, 128, 2)) || tsp::meet(tsp::runs_of(k.data, 4096), tsp::runs_of(q, n, 16, 128, 2))) return 4;
    std::printf("overlap_check: ok, %d meet, %d interleave, %d apart\n", met, interleaved, apart);
    return met > 1000 && interleaved > 1000 && apart > 1000 ? 0 : 5;
}
