// The height of the persistent kernel's tiles in gg_gemm_i8. Host code alone, without HIP, so that tests/i8_choice.cpp
// holds measured problems to it.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace gg {

// M-tiles of `tile_m` rows that `rows` rows in groups of unknown sizes are expected to fill: the last tile of a group is
// half full on average, whatever the load, and a group has one tile at least. One group is known.
inline double expected_tiles(int group_num, int64_t rows, int tile_m) {
    if (group_num == 1)
        return double((rows + tile_m - 1) / tile_m);
    const double groups = double(std::min<int64_t>(group_num, rows));
    return std::max(groups, double(rows) / tile_m + 0.5 * groups);
}

// Whether tiles of 192 rows are taken where 256 fit. A K step of one takes kShortStep of the taller tile's, so they pay where
// they need no more rounds of workgroups (and not where the GPU is full of rows: every byte of w is staged for fewer of
// them). The count of tiles is sure to about n_tiles sqrt(groups / 12), the spread of the groups' last tiles: rounds are
// averaged over three counts that far apart, and a gain of 5 % on average is taken if the worst case loses no more than 12 %.
//
// Measured with 133 problems of 1 to 64 groups of 64 to 3000 rows on average, each under seven loads (equal groups, near
// equal ones, gamma distributions of shape 6 and 1, every other group empty, one group with half of the rows, 1 / rank);
// geometric mean of the time over the better height's, and the worst: this rule 1.016, 1.42; 256 rows always 1.087, 1.26;
// 192 always 1.033, 1.57. By load 1.020, 1.016, 1.012, 1.011, 1.026, 1.018, 1.014; 35 of 1209 lose over 15 %. (The tiles
// expected of a gamma distribution of shape 6, by its octiles: 1.018, 1.32, 46; of an exponential one 1.015, 1.43.)
// us, 256 and 192 rows: taken 8 groups of 4160 rows in all, 7168 x 2048 71-82 and 66-70 (1 / rank 61, 68); the same, 4096 x
// 7168 136-153, 119-136; 8320 rows 217-233, 192-208; 1200 65-82, 62-74; left 32 of 16640, 2880 x 2880 156-182, 162-186;
// missed 64 of 8192, 2048 x 1408 50-67, 48-60; wrong for 9 of 1200, 7488 x 4672 with every other group empty 67, 95 (other
// loads 117-128, 106-116).
constexpr double kShortStep = 0.83;
inline bool short_tiles_pay(int group_num, int64_t rows, int64_t n_tiles, int cus) {
    constexpr int kTall = 256, kShort = 192;
    const auto rounds = [&](int tile_m, double *all) { // on average; all: of the three counts
        const double tiles  = expected_tiles(group_num, rows, tile_m) * n_tiles;
        const double spread = group_num == 1 ? 0.0
                                             : std::sqrt(group_num / 12.0) * std::min(1.0, double(rows) / group_num / tile_m) * n_tiles;
        for (int i = 0; i < 3; ++i)
            all[i] = std::max(1.0, std::ceil((tiles + 1.22 * (i - 1) * spread) / cus));
        return (all[0] + all[1] + all[2]) / 3;
    };
    double       tall[3], low[3];
    const double t = rounds(kTall, tall), s = rounds(kShort, low);
    return kShortStep * s < 0.95 * t && kShortStep * low[2] < 1.12 * tall[0];
}

} // namespace gg
