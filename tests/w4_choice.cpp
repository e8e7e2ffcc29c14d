// The kernel that gg_gemm_w4 takes for "groups rows columns" triples on the command line, one name a line.
#include <cstdio>
#include <cstdlib>

#include "gg_w4_choice.h"

int main(int argc, char **argv) {
    static const char *names[] = {"few64", "few32", "few16", "rows"};
    for (int i = 1; i + 2 < argc; i += 3)
        std::puts(names[static_cast<int>(gg::layer::w4_choice(std::atoll(argv[i]), std::atoll(argv[i + 1]), std::atoll(argv[i + 2])))]);
    return 0;
}
