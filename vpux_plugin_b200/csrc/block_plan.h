// Which rows an expert of a grouped product owns, how many tiles that can make, and which form of the product runs: plain functions
// that the kernels, the host side and the tests share.
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

// ---- the forms of the product on the tensor cores -------------------------------------------------------------------------
// SwapN: the weights are the 128-row operand, N activations the other one, column blocks shared in clusters. WideN: 128 activations by N outputs.
enum class Form { Swap16, Swap32, Swap128, Wide128, Wide256 };

// The form goes by the rows of activations (of an expert, on average) and by the tiles that there are. Times in us of short bursts
// replayed from a graph (the power limit slows both sides of a long run alike), [rows, outputs, columns]:
//   up to 16 rows       [16, 4096, 4096]     Swap16 6.5   Swap32 6.9   Swap128 9.4
//   up to 32            [32, 11008, 4096]    Swap16 13.7  Swap32 11.7  Swap128 19.4; grouped, 32 rows on average, 16 experts [2048, 2048]:
//                                            Swap32 19.4  Wide128 17.0  Wide256 16.8, since most experts' rows end inside a tile
//   up to 64, where tiles of 128 x 128 leave half of the multiprocessors idle:
//                       [64, 4096, 4096]     Swap32 8.3   Swap128 9.6  ([65, 4096, 4096] Wide128 10.8); else
//                       [64, 11008, 4096]    Swap32 16.4  Swap128 19.9 ([65, 11008, 4096] Wide128 13.1)
//   above, where they leave three quarters idle:
//                       [512, 1024, 8192]    Swap128 14.7  Wide128 18.6  Wide256 26.2; else
//                       [192, 4096, 4096]    Swap128 14.9  Wide128 11.1  Wide256 15.5
//   and the rest by the rounds that the tiles take; one of Wide256's takes 1.65 times as long as one of Wide128's:
//                       [512, 4096, 4096]    128 or 64 tiles, one round either way   Wide128 11.8  Wide256 16.7
//                       [1024, 4096, 4096]   256 or 128 tiles, two rounds or one     Wide128 20.7  Wide256 18.6
//                       [1500, 4096, 4096]   three rounds or two                     Wide128 29.8  Wide256 31.8
//                       [4096, 11008, 4096]  nineteen or ten                         Wide128 191.9 Wide256 163.7
inline Form form_of(int64_t x_rows, int64_t experts, int64_t outputs, int64_t sms) {
    const int64_t rows = experts ? (x_rows + experts - 1) / experts : x_rows;
    // (of the experts' last tiles, half are counted: the bound that the grid is sized by counts one for every expert)
    const int64_t row_tiles = (x_rows + 127) / 128 + experts / 2;
    const int64_t few = row_tiles * ((outputs + 127) / 128), wide = row_tiles * ((outputs + 255) / 256);
    if (rows <= 16) return Form::Swap16;
    if (rows <= 32 && !experts) return Form::Swap32;
    if (rows <= 64 && few * 2 <= sms) return Form::Swap32;
    if (few * 4 <= sms) return Form::Swap128;
    if ((wide + sms - 1) / sms * 165 < (few + sms - 1) / sms * 100) return Form::Wide256;
    return Form::Wide128;
}

// Few rows: CTAs that share a tile's column blocks, where every tile can have a cluster of its own. A CTA's time goes with the column
// blocks that it walks through one after the other, whether another CTA shares its multiprocessor or not; joining costs
// about as much as four of them. In us by CTAs per cluster, the rule's choice marked (the same bursts; "more" than there is room for):
//   Swap16   [1, 4096, 4096]      1: 10.1  2: 7.3   3: 6.4   4: 6.1   6: 6.0   8: 6.3 *
//            [1, 11008, 4096]     1: 12.6  2: 11.9  3: 10.1 *  4: 14.4 more  8: 18.1 more
//            [16, 4096, 11008]    1: 22.7  2: 15.2  4: 11.7  6: 11.3  8: 10.9 *
//   Swap32   [48, 4096, 11008]    1: 31.5  2: 20.1  3: 15.8  4: 14.0 *  5: 21.1 more  8: 19.7 more
//            [64, 1024, 8192]     1: 20.3  2: 12.9  4: 9.3   8: 7.5 *
//   Swap128  [256, 1024, 8192]    1: 32.3  2: 20.9  4: 13.7 *  8: 20.1 (clusters of eight CTAs with a multiprocessor each wait more often)
//   per_sm    CTAs that a multiprocessor holds
//   fours     groups of four columns in a tile; the CTAs of a cluster own them in turn, and `places` bounds what all of them keep
inline int ranks_of(int64_t tiles, int64_t col_blocks, int per_sm, int64_t sms, int fours, int places) {
    int best = 1;
    int64_t least = col_blocks;
    for (int r = 2; r <= 4 * per_sm && 2 * r <= col_blocks && tiles * r <= per_sm * sms; ++r) {
        const int64_t load = (col_blocks + r - 1) / r + 4;
        if ((fours + r - 1) / r * r <= places && load < least) {
            least = load;
            best = r;
        }
    }
    return best;
}

}  // namespace vf
