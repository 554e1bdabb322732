// Which rows the experts of a grouped product get from their offsets (csrc/block_plan.h), restated for a warp that reads 32 experts
// at a time as the kernels do, over offsets that keep the rules and offsets that break them in every way. Needs no device.
#include <cstdio>
#include <random>
#include <vector>

#include "block_plan.h"

namespace {

int failed = 0;

#define CHECK(c)                                            \
    do {                                                    \
        if (!(c)) {                                         \
            std::printf("line %d: %s\n", __LINE__, #c);     \
            ++failed;                                       \
        }                                                   \
    } while (0)

struct Walked {
    std::vector<vf::RowRange> ranges;
    bool moved = false;
};

// Groups of 32: one vote whether all of them keep the rules, else the maximum over the lanes in front (five doubling steps)
Walked by_warps(const std::vector<int64_t>& offs, int64_t rows) {
    Walked w;
    const int experts = int(offs.size()) - 1;
    int reach = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
        int64_t a[32], b[32];
        int lo[32], hi[32], to[32];
        bool in[32], ok = true;
        for (int l = 0; l < 32; ++l) {
            in[l] = e0 + l < experts;
            a[l] = in[l] ? offs[size_t(e0 + l)] : 0;
            b[l] = in[l] ? offs[size_t(e0 + l + 1)] : 0;
            lo[l] = int(a[l]);
            hi[l] = int(b[l]);
        }
        for (int l = 0; l < 32; ++l) ok = ok && (!in[l] || (a[l] >= 0 && a[l] <= b[l] && b[l] <= rows && lo[l] >= (l ? hi[l - 1] : reach)));
        if (ok) {
            reach = hi[31];
        } else {
            for (int l = 0; l < 32; ++l) to[l] = std::max(reach, in[l] ? vf::row_reach(a[l], b[l], rows) : 0);
            for (int d = 1; d < 32; d <<= 1)
                for (int l = 31; l >= d; --l) to[l] = std::max(to[l], to[l - d]);
            for (int l = 0; l < 32; ++l) {
                const vf::RowRange r = vf::rows_of(a[l], b[l], rows, l ? to[l - 1] : reach);
                w.moved = w.moved || (in[l] && r.moved);
                lo[l] = in[l] ? r.lo : 0;
                hi[l] = in[l] ? r.hi : 0;
            }
            reach = to[31];
        }
        for (int l = 0; l < 32 && in[l]; ++l) w.ranges.push_back({lo[l], hi[l], false});
    }
    return w;
}

void check(const std::vector<int64_t>& offs, int64_t rows) {
    const int experts = int(offs.size()) - 1;
    bool keep = offs[0] >= 0 && offs.back() <= rows;
    for (int e = 0; e < experts; ++e) keep = keep && offs[size_t(e)] <= offs[size_t(e) + 1];
    const Walked w = by_warps(offs, rows);
    CHECK(w.moved == !keep);
    CHECK(int(w.ranges.size()) == experts);
    int end = 0, reach = 0;
    for (int e = 0; e < experts; ++e) {
        const vf::RowRange r = w.ranges[size_t(e)];
        CHECK(r.lo >= end && r.hi >= r.lo && r.hi <= rows);  // disjoint, ascending, inside
        end = r.hi;
        const vf::RowRange one = vf::rows_of(offs[size_t(e)], offs[size_t(e) + 1], rows, reach);  // one expert after the other
        CHECK(one.lo == r.lo && one.hi == r.hi);
        reach = one.hi;
        if (keep) CHECK(r.lo == offs[size_t(e)] && r.hi == offs[size_t(e) + 1]);
    }
    for (int bm : {16, 32, 64, 128}) {
        int64_t tiles = 0;
        for (const vf::RowRange& r : w.ranges) tiles += vf::tiles_of_rows(r.lo, r.hi, bm);
        CHECK(tiles <= vf::most_row_tiles(rows, experts, bm));
    }
}

}  // namespace

int main() {
    // an expert behind a decrease began again at a small row: 9 tiles of 16 rows where at most 8 can be
    check({0, 48, 0, 48, 0, 48}, 48);
    check({0, 128, 0, 128, 0, 128, 0, 128, 0}, 128);
    check({0, 30, 20, 40}, 40);
    check({50, 60, 70, 80}, 40);
    check({0, 10, int64_t(1) << 40, int64_t(1) << 41}, 40);
    check({-(int64_t(1) << 62), -3, -2, -1}, 40);
    check({INT64_MIN, INT64_MAX, INT64_MIN, INT64_MAX}, INT32_MAX - 256);
    check({0, (int64_t(1) << 32) + 5, 7}, 40);  // equal to good offsets in their low 32 bits
    check({0, 0, 7, 7, 40}, 40);
    std::mt19937_64 rng(5);
    for (int turn = 0; turn < 20000; ++turn) {
        const int64_t rows = turn % 5 == 0 ? INT32_MAX - 256 : 1 + int64_t(rng() % 3000);
        std::vector<int64_t> offs(2 + rng() % (turn % 3 ? 8 : 150));
        const int kind = turn % 7;
        for (size_t e = 0; e < offs.size(); ++e) {
            const int64_t any = int64_t(rng() % uint64_t(rows + 1));
            offs[e] = kind == 0 ? int64_t(rng())                                                  // memory that nobody wrote
                    : kind == 1 ? (e & 1 ? rows : 0)                                              // up and down
                    : kind == 2 ? rows - int64_t(e) * rows / int64_t(offs.size())                 // down
                    : kind == 3 ? any * 2 - rows / 2                                              // some outside
                                : any;
        }
        if (kind >= 4) std::sort(offs.begin(), offs.end());
        if (kind == 5) offs[rng() % offs.size()] = int64_t(rng() % uint64_t(rows + 1));             // one out of order
        if (kind == 6) offs[rng() % offs.size()] += int64_t(rng() % 3) - 1;                          // off by one
        check(offs, rows);
    }
    std::printf("block plan: %d failed\n", failed);
    return failed != 0;
}
