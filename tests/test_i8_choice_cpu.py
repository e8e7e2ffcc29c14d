"""gg_gemm_i8's choice between tiles of 256 and 192 rows, which knows the number of rows but not their groups' sizes."""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


@pytest.fixture(scope="module")
def choice(tmp_path_factory):
    exe = tmp_path_factory.mktemp("i8") / "i8_choice"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "groupgemm-cktile-optimized_amd", "csrc"),
                    os.path.join(ROOT, "tests", "i8_choice.cpp"), "-o", str(exe)], check=True)

    def run(what, cases):
        r = subprocess.run([str(exe), what] + [str(v) for c in cases for v in c], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0
        return [float(v) for v in r.stdout.split()]

    return run


def _loads(groups, rows):
    """Sizes of the groups: equal, spread evenly, and as exponentials fall."""
    r = random.Random(groups * 1000003 + rows)
    for share in ([1.0] * groups, [r.uniform(0.3, 1.7) for _ in range(groups)], [r.expovariate(1.0) for _ in range(groups)]):
        yield [int(rows * s / sum(share)) for s in share]


@pytest.mark.parametrize("tile_m", [192, 256])
@pytest.mark.parametrize("groups", [2, 3, 8, 21, 64])
def test_expected_tiles_hold_the_rows_of_any_load(choice, groups, tile_m):
    averages = [1, 40, 100, 191, 192, 257, 500, 1000, 4000, 30000, 100000]
    got = choice("tiles", [(groups, groups * a, tile_m) for a in averages])
    for a, tiles in zip(averages, got):
        assert tiles * tile_m >= groups * a and tiles >= groups  # as many rows as there are, a tile for each group
        assert tiles <= groups * (a / tile_m + 1)
        if a >= 4 * tile_m:  # half a tile a group off from any load at most, as the last tile of a group is between empty and full
            for sizes in _loads(groups, groups * a):
                assert abs(sum(-(-s // tile_m) for s in sizes) - tiles) <= 0.55 * groups + 1, (a, sizes)


def test_one_group_has_its_tiles(choice):
    assert choice("tiles", [(1, 193, 192), (1, 192, 192), (1, 2048, 256), (1, 5, 256)]) == [2, 1, 8, 1]


# us on 256- and on 192-row tiles under seven loads (equal, near equal, two spreads, half of the groups empty, one with half
# of the rows, 1 / rank): those of which all but one gain or lose 5 % and more
TAKEN = [(8, 4160, 7168, 2048), (8, 8320, 4096, 7168), (8, 1200, 4096, 7168), (9, 1200, 7488, 4672), (13, 3622, 3520, 2496),
         (2, 683, 5184, 640), (25, 1774, 3392, 3520), (19, 20803, 512, 576), (3, 7252, 2816, 3200)]
LEFT = [(32, 16640, 2880, 2880), (35, 101422, 4736, 768), (14, 25279, 2880, 3584), (38, 57286, 1664, 3520), (4, 3573, 10240, 5056)]


def test_measured_choices(choice):
    assert choice("short", TAKEN) == [1] * len(TAKEN) and choice("short", LEFT) == [0] * len(LEFT)
