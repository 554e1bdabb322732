// Which rows an expert of a grouped product owns and how many tiles that can make: plain functions that the kernels, the host
// side and the tests without a device share.
#pragma once

#include <algorithm>
#include <cstdint>

#ifdef __CUDACC__
#define VF_BOTH __host__ __device__ __forceinline__
#else
#define VF_BOTH inline
#endif

namespace vf {

// Expert e owns rows offsets[e] .. offsets[e + 1]. Offsets that decrease or leave the operand are moved so that an expert's rows
// never begin before those of the experts in front of it end. Ranges are therefore disjoint and ascending whatever the
// offsets hold, no row is written twice, and most_row_tiles() bounds what a walk over them finds.
struct RowRange {
    int lo, hi;
    bool moved;  // the offsets break the rules
};

VF_BOTH int row_within(int64_t v, int64_t rows) {
    return int(v < 0 ? 0 : (v > rows ? rows : v));
}
// How far an expert's own offsets reach; the maximum over all experts up to e is where the range of e ends
VF_BOTH int row_reach(int64_t a, int64_t b, int64_t rows) {
    const int x = row_within(a, rows), y = row_within(b, rows);
    return x > y ? x : y;
}
// The range of an expert with offsets a and b behind experts that reach to `reach`
VF_BOTH RowRange rows_of(int64_t a, int64_t b, int64_t rows, int reach) {
    RowRange r;
    const int x = row_within(a, rows), y = row_within(b, rows);
    r.lo = x > reach ? x : reach;
    r.hi = y > r.lo ? y : r.lo;
    r.moved = r.lo != a || r.hi != b;
    return r;
}

VF_BOTH int tiles_of_rows(int lo, int hi, int bm) {
    return int(uint32_t(hi - lo + bm - 1) / uint32_t(bm));
}

// Row tiles of `bm` rows: exact for one group (experts = 0); for experts an upper bound, since each may end inside a tile.
inline int64_t most_row_tiles(int64_t rows, int64_t experts, int bm) {
    const int64_t whole = (rows + bm - 1) / bm;
    return experts ? std::min(rows, whole + experts) : whole;
}

// Tiles are counted in 32 bits, and so is one step of the grid (at most a few thousand) behind the last of them. Whichever form runs,
// its tiles are not smaller than 16 rows by 64 columns, so a product below this limit by those is counted right by all.
constexpr int64_t kTileLimit = (int64_t(1) << 31) - (int64_t(1) << 20);

inline bool too_many_tiles(int64_t rows, int64_t experts, int64_t outputs) {
    const int64_t cols = (outputs + 63) / 64;
    return cols && most_row_tiles(rows, experts, 16) > kTileLimit / cols;
}

}  // namespace vf
