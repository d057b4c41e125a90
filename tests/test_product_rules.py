"""Where the blocks of the products of any shape work (csrc/product_launch.h), on the host alone."""
import ctypes as C
import subprocess
from collections import Counter
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
XCDS, UNITS = 8, 256  # block b runs on XCD b % 8, which has 32 units


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    library = tmp_path_factory.mktemp("rules") / "libproduct.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", str(ROOT / "tests/product_rules.cpp"), "-o", str(library)], check=True)
    return C.CDLL(str(library))


def test_few_blocks_are_shared_out_over_the_xcds(rules):
    """Up to 256 tiles go to one unit each: every tile to one block, and no XCD has more than one block above any other's."""
    out = (C.c_int * 2)()
    for tiles_m in range(1, UNITS + 1):
        for tiles_n in range(1, UNITS // tiles_m + 1):
            seen, busy = set(), Counter({xcd: 0 for xcd in range(XCDS)})
            for block in range(tiles_m * tiles_n):
                rules.product_few_place(block, tiles_m, tiles_n, out)
                m, n = out
                assert 0 <= m < tiles_m and 0 <= n < tiles_n and (m, n) not in seen
                seen.add((m, n))
                busy[block % XCDS] += 1
            assert max(busy.values()) - min(busy.values()) <= 1, (tiles_m, tiles_n, dict(busy))


@pytest.mark.parametrize("grid", [1, 7, 8, 9, 200, 256, 511, 512])
def test_first_tiles_are_a_permutation(rules, grid):
    tiles = [rules.product_first_tile(block, grid) for block in range(grid)]
    assert sorted(tiles) == list(range(grid))
    for block in range(grid - 8):
        assert tiles[block + 8] == tiles[block] + 1
