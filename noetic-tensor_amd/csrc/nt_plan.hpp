// How a product [m, k] x [n, k] is cut up: the tile (nt_tile.hpp) and the splits of k, by what they cost.
#pragma once

#include <cstdint>

namespace nt {
namespace tile {

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// A workgroup's tile: 32 TM WM rows by 128 WN columns. A wave takes 128 columns whatever the tile, so that the
// readout's sums over a row are in the same order whatever rows are scored with it.
template <int TM_, int WM_, int WN_>
struct Shape {
    static constexpr int TM = TM_, TN = 4, WM = WM_, WN = WN_;
    static constexpr int kThreads = 64 * WM * WN, kRows = 32 * TM * WM, kCols = 128 * WN;
};
typedef Shape<4, 2, 2> Large;   // 256 x 256, a workgroup a CU
typedef Shape<1, 4, 1> Medium;  // 128 x 128, two workgroups a CU: one's output while the other multiplies
typedef Shape<1, 2, 1> Small;   // 64 x 128, two workgroups of two waves a CU

enum class Size { kSmall, kMedium, kLarge };
struct Plan {
    Size size;
    int64_t per, splits;  // bytes of k of a split (a row's), a multiple of 64
    double cost;          // us
};

// The tile of the least cost for `kb` bytes of k, split where `split` allows it: rounds of the workgroups that run
// at once, each its stages of 64 bytes and its output. Measured (us a stage, a round full): 0.92, 0.57 and 0.36 for
// Large, Medium and Small, or 0.33 and 0.25 in a round of one workgroup a CU; an output of Large about 6 us, of
// Medium and Small less than their share of it, since it goes on beside the other workgroup's products; the slabs of a
// split k 4 us, 0.15 a slab and their bytes, written and read, at 4 TB/s. So 4096 x 128256 takes Large, 333 x 50257 x 1001 Medium (a
// pass over the logits 99 -> 77 us), 64 rows Small (29 -> 16 us at 32000 x 1024).
inline Plan plan(int64_t m, int64_t n, int64_t kb, bool split) {
    if (kb < 64) kb = 64;
    struct Kind {
        Size size;
        int64_t rows, cols, slots;
        double stage, alone, output;
    };
    static const Kind kinds[] = {{Size::kLarge, Large::kRows, Large::kCols, 256, 0.92, 0.92, 6.0},
                                 {Size::kMedium, Medium::kRows, Medium::kCols, 512, 0.57, 0.33, 2.5},
                                 {Size::kSmall, Small::kRows, Small::kCols, 512, 0.36, 0.25, 1.5}};
    Plan best{};
    for (const Kind &c : kinds) {
        const int64_t tiles = ceil_div(m, c.rows) * ceil_div(n, c.cols);
        for (int64_t r = 0; r <= 4; r++) {  // unsplit, and the splits that give every CU one to four workgroups
            int64_t s = r == 0 ? 1 : 256 * r / tiles;
            s = s > 64 ? 64 : s;
            // (512 bytes of k a split at the least: 8-bit products of 64 x 1000 x 8192 29 -> 10 us, 16 x 256 x 16384 52 -> 8)
            s = s > 1 && s > kb / 512 ? kb / 512 : s;
            if (s < 1 || (s > 1 && !split)) continue;
            const int64_t per = round_up(ceil_div(kb, s), 64), splits = ceil_div(kb, per);
            const int64_t wgs = tiles * splits, rounds = ceil_div(wgs, c.slots);
            const double cost = double(rounds) * (double(per / 64) * (wgs <= 256 ? c.alone : c.stage) + c.output) +
                                (splits > 1 ? 4.0 + double(splits) * (0.15 + double(m) * double(n) * 8e-6 / 4.0) : 0.0);
            if (best.per == 0 || cost < best.cost) best = Plan{c.size, per, splits, cost};
        }
    }
    return best;
}

// The columns of [m, n] that go by Large tiles in whole rounds of 256, where the rest by itself costs less than
// one more round of them does (a multiple of a tile's; 0: no such split). 2048 x 50304 is 1576 tiles: 1536, and the
// last 1152 columns apart (a pass over the logits of dim 4096 828 -> 787 us).
inline int64_t whole_rounds(int64_t m, int64_t n, int64_t kb) {
    const Plan all = plan(m, n, kb, false);
    if (all.size != Size::kLarge) return 0;
    const int64_t tm = ceil_div(m, Large::kRows), tiles = tm * ceil_div(n, Large::kCols);
    const int64_t cols = tiles / 256 * 256 / tm * Large::kCols;
    if (cols <= 0 || cols >= n) return 0;
    return plan(m, cols, kb, false).cost + plan(m, n - cols, kb, false).cost + 4.0 < all.cost ? cols : 0;
}

}  // namespace tile
}  // namespace nt
