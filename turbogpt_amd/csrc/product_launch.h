// Which kernel of product_tile.h and product_few.h takes a product, and where its blocks work: plain functions of a call's shape.
#pragma once
#include <cstdint>

namespace product {

// A block's first tile, in the order in which tiles are walked: a block's neighbours in its XCD (blocks 8 apart) take neighbouring tiles, which share
// rows of a and b in that XCD's L2, and every XCD has as many tiles as any other, or one more.
constexpr int first_tile(int block, int grid) {
    const int each = grid >> 3, rest = grid & 7, xcd = block & 7;
    return xcd * each + (xcd < rest ? xcd : rest) + (block >> 3);
}

struct Place {
    int m, n; // in tiles
};
// product_few.h: a block a tile, column by column, so that neighbours share their rows of b.  With a column's blocks all in one XCD, results of few columns
// left the others idle: 8 bits, K = 1024, 6400 x 128 22.5 us, now 7.7; 16384 x 64 41, now 9.3; gated, 4096 x 64, D = 1024 20.9, now 8.
constexpr Place few_place(int block, int tiles_m, int tiles_n) {
    const int tile = first_tile(block, tiles_m * tiles_n);
    return {tile % tiles_m, tile / tiles_m};
}

// Which kernel.  While 256 blocks, one a unit, cover the result, the smallest of the few kernel's shapes that does it (its blocks share out k, so one
// is never worse than more: 1000 columns, K = 1904 in 8 bits, 1024 rows 11.3 us, tiles of 64 x 128 14.3; at 2048 rows, 512 blocks, 18 and 15.2).
// Otherwise the least of the tiles' estimated times, us: per stage a tile's time alone on its unit, or of two (of 256 x 256 it grows with the
// share of units that have one, as all of them ask the same memory), and an epilogue; fitted to the operators at 64 to 16384 rows, by what they choose: a
// pass by itself may take longer (gated, 333 rows, 1720 columns, D = 640 on 64 x 128: 8.4, estimated 5.7).  Gated, 2 x 2816
// columns, D = 1024, on 64 x 128, 128 x 128, 256 x 256: 512 rows 15.8, 17.7, 26; 1024 28.9, 20.7, 27.5; 2048 40, 40, 30.
enum ProductKernel { FEW_16, FEW_32, FEW_64x32, FEW_64, TILES_64x128, TILES_128, TILES_256 };
// how many blocks of a kernel of tiles are at work at a time, on 256 units
constexpr int most_blocks(ProductKernel kernel) {
    return kernel == TILES_256 ? 256 : 512;
}
struct TileTimes {
    double alone, two, epilogue;
};
inline double tiles_us(int64_t tiles, int stages, const TileTimes &t) {
    const int64_t rounds = tiles / 512, rest = tiles % 512;
    return rounds * (stages * t.two + t.epilogue) + (rest > 256 ? stages * t.two + t.epilogue : rest ? stages * t.alone + t.epilogue : 0.0);
}
inline double large_tiles_us(int64_t tiles, int stages, const TileTimes &t) { // `two`: alone, with every unit at work
    const int64_t rounds = tiles / 256, rest = tiles % 256;
    return rounds * (stages * t.two + t.epilogue) + (rest ? stages * (t.alone + (t.two - t.alone) * (rounds ? 1.0 : rest / 256.0)) + t.epilogue : 0.0);
}
// M and N: of the result; gated: N columns of either matrix, and no FEW_64
inline ProductKernel product_kernel(int M, int N, int stages, bool e4m3, bool gated) {
    const auto count = [&](int rows, int columns) { return (int64_t(M) + rows - 1) / rows * ((int64_t(N) + columns - 1) / columns); };
    if (count(16, 16) <= 256)
        return FEW_16;
    if (count(32, 32) <= 256)
        return FEW_32;
    if (count(64, 32) <= 256)
        return FEW_64x32;
    if (!gated && count(64, 64) <= 256)
        return FEW_64;
    const int of = gated ? 2 : 1; // a tile's columns of B for one of the result
    const double low = tiles_us(count(64, 128 / of), stages, e4m3 ? TileTimes{0.54, 0.90, 1.5} : TileTimes{0.42, 0.72, 1.5});
    const double square = tiles_us(count(128, 128 / of), stages, e4m3 ? TileTimes{0.77, 1.25, 2.5} : TileTimes{0.57, 1.10, 2.5});
    const double large = large_tiles_us(count(256, 256 / of), stages, e4m3 ? TileTimes{1.65, 1.90, 6.0} : TileTimes{0.95, 1.58, 6.0});
    if (large <= low && large <= square)
        return TILES_256;
    return square <= low ? TILES_128 : TILES_64x128;
}

} // namespace product
