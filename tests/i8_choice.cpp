// "tiles" groups rows tile_m, ..: the M-tiles that gg_gemm_i8 expects; "short" groups rows n k, ..: 1 where it takes
// 192-row tiles on 256 CUs. One number a line.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "gg_i8_choice.h"

int main(int argc, char **argv) {
    const bool tiles = argc > 1 && std::strcmp(argv[1], "tiles") == 0;
    for (int i = 2; i + (tiles ? 2 : 3) < argc; i += tiles ? 3 : 4) {
        const long long groups = std::atoll(argv[i]), rows = std::atoll(argv[i + 1]), n = std::atoll(argv[i + 2]);
        if (tiles)
            std::printf("%.9g\n", gg::expected_tiles(static_cast<int>(groups), rows, static_cast<int>(n)));
        else
            std::printf("%d\n", gg::short_tiles_pay(static_cast<int>(groups), rows, (n + 255) / 256, 256));
    }
    return 0;
}
