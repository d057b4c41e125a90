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


FEW = ("FEW_16", "FEW_32", "FEW_64x32", "FEW_64")
TILES = {"TILES_64x128": (64, 128), "TILES_128": (128, 128), "TILES_256": (256, 256)}
KERNELS = (*FEW, *TILES)


def features(rules, operator, M, N, stages, e4m3=False, is_gated=False):
    """What a product of M x N results runs: the kernel, and of a kernel of tiles whether its blocks take one or many, and whether a tile has a single stage."""
    index = rules.product_kernel_of(M, N, stages, e4m3, is_gated)
    name = KERNELS[index]
    found = {(operator, name)}
    if name in TILES:
        rows, columns = TILES[name]
        tiles = -(-M // rows) * -(-N // (columns // 2 if is_gated else columns))
        found.add((operator, name, "many" if tiles > rules.product_most_blocks(index) else "one"))
        if stages == 1:
            found.add((operator, name, "a stage"))
    return found


def gated_features(rules, M, F, D):
    stages = -(-D // 64)
    found = features(rules, "H", M, F, stages, is_gated=True) | features(rules, "dH", M, F, stages)
    if not (M % 128 == 0 and M >= 1024 and (D % 128 == 0 or D % 192 == 0) and F % 16 == 0):  # the framework's product otherwise
        found |= features(rules, "dX", M, D, -(-2 * F // 64))
    return found


def test_every_kernel_is_compared_with_the_definition(rules):
    """Every (operator, kernel) that a shape can reach is reached by a shape of the tests against 64 bits: they run both activations, with and without kept
    pre-activations, with and without a residual."""
    import test_gpu_gated
    import test_gpu_gemm_q8
    import test_gpu_product_kernels as more
    tested = set()
    for shape in test_gpu_gated.SHAPES + more.GATED:
        tested |= gated_features(rules, *shape)
    for M, N, K in test_gpu_gemm_q8.SHAPES + more.Q8:
        tested |= features(rules, "Y", M, N, -(-K // 128), e4m3=True)
    wanted = {(operator, name) for operator in ("H", "dH", "dX", "Y") for name in KERNELS if (operator, name) != ("H", "FEW_64")}
    wanted |= {(operator, name, how) for operator in ("H", "dH", "dX", "Y") for name in TILES for how in ("one", "many")}
    # the rule gives 256 x 256 tiles no product of one stage
    wanted |= {(operator, name, "a stage") for operator in ("H", "dH", "dX", "Y") for name in ("TILES_64x128", "TILES_128")}
    assert wanted <= tested, sorted(wanted - tested)
    assert not any(name == "TILES_256" and rest == ["a stage"] for _, name, *rest in tested)


def test_products_of_one_stage_have_no_tiles_of_256(rules):
    for M in (1, 100, 1000, 4096, 16384, 100000, 1 << 20):
        for N in (8, 128, 1000, 4096, 1 << 16):
            for e4m3, is_gated in ((0, 0), (0, 1), (1, 0)):
                assert KERNELS[rules.product_kernel_of(M, N, 1, e4m3, is_gated)] != "TILES_256"
