// Where the blocks of the products of any shape work, for tests without a GPU.
#include "../turbogpt_amd/csrc/product_launch.h"

extern "C" {
void product_few_place(int block, int tiles_m, int tiles_n, int *out) {
    const product::Place p = product::few_place(block, tiles_m, tiles_n);
    out[0] = p.m, out[1] = p.n;
}
int product_first_tile(int block, int grid) {
    return product::first_tile(block, grid);
}
}
