// Where the blocks of product_tile.h and product_few.h work: plain functions of a call's shape, on the device and on the host alike.
#pragma once

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

} // namespace product
