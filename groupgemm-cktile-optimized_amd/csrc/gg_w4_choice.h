// Which kernel a call of gg_gemm_w4 takes. Host code alone, without HIP, so that tests/w4_choice.cpp holds the tests'
// sizes to it.
#pragma once

#include <algorithm>
#include <cstdint>

namespace gg {
namespace layer {

// How many pieces of `rows` rows the groups have at most, where they lie inside x and do not overlap.
inline int64_t w4_pieces(int64_t group_num, int64_t total_m, int rows) {
    return std::max<int64_t>(1, std::min(group_num, total_m) + total_m / rows);
}

// The few-row instances of 64, 32 and 16 columns a workgroup, and the many-row one.
enum class W4Choice { kFew64, kFew32, kFew16, kRows };

// The instance by the rows that a group has on average and the workgroups there are. Measured (us; few-row instances of
// 64, 32 and 16 columns a workgroup, then the many-row one, of 32 rows and 128 columns):
//   rows per group (ragged; 32 groups of 2880 x 2880, k of a scale 32, zero points / 16 of 4096 x 4096, 128):
//     8: 44.6, 54.6, 82.4, 47.4 / 32.5, 42.0, 57.4, 40.5          12: 50.1, 63.2, 100.9, 49.3 / 36.8, 48.7, 70.7, 38.0
//     16: 54.5, 70.8, 114.9, 52.8 / 40.3, 56.1, 84.6, 41.6        20: 66.0, 84.0, 138.2, 58.9 / 49.0, 68.7, 104.7, 47.6
//     24: 71.8, 95.5, 157.6, 65.2 / 52.7, 74.3, 118.0, 48.3       48: 120.1, 162.1, 269.7, 98.5 / 87.3, 133.5, 221.8, 63.1
//     16 rows in every group of the first: 45.0, 60.3, 100.5, 50.0; 24: 71.0, 94.2, 157.3, 51.0
//   Many-row instances of 16, 48 and 64 rows, or of 64, 192 and 256 columns, gain 3 to 17 % where their sizes fit and
//   lose 5 to 50 % elsewhere.
//   workgroups of 64 columns (one row): 8 of 512 x 7168: 11.9, 7.3, 6.1; 32 of 512 x 2048: 6.3, 5.0, 4.6; 128 of
//     4096 x 1024: 5.2, 4.7, 5.5; 224 of 14336 x 4096: 10.8, 9.5, 12.0; 448 of 7168 x 2048: 9.7, 11.9, 13.8; 4 groups of 20
//     rows, 2048 x 4096 (288): 11.6, 13.7, 18.8
//   the many-row one does not split k: with few workgroups it loses (64-column few-row and many-row instance; workgroups of the
//     latter): 160 of 24 rows, 4096 x 4096 17.6, 26.8; 320 27.5, 30.8 (k 9600: 63.7, 75.8; 1024: 12.2, 11.2); 448 of 14336 x
//     4096 41.3, 34.6; 510 of 1280 x 5120 60.0, 50.5. Half a piece for each group and the rows / 32: about as many as there are.
inline W4Choice w4_choice(int64_t group_num, int64_t total_m, int64_t n) {
    const int64_t tiles = (n + 15) / 16, slots = std::max<int64_t>(1, std::min(group_num, total_m)), per = total_m / slots;
    const int64_t wide = (tiles + 7) / 8 * (slots + total_m / 16) / 2, narrow = (tiles + 3) / 4 * w4_pieces(group_num, total_m, 16);
    return per > 16 && wide >= 384 ? W4Choice::kRows
           : narrow >= 256          ? W4Choice::kFew64
           : narrow >= 64           ? W4Choice::kFew32
                                    : W4Choice::kFew16;
}

} // namespace layer
} // namespace gg
