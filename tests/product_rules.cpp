// Which kernel takes a product of any shape and where its blocks work, for tests without a GPU.
#include "../turbogpt_amd/csrc/product_launch.h"

extern "C" {
int product_kernel_of(int M, int N, int stages, int e4m3, int gated) {
    return product::product_kernel(M, N, stages, e4m3, gated);
}
int product_most_blocks(int kernel) {
    return product::most_blocks(product::ProductKernel(kernel));
}
void product_few_place(int block, int tiles_m, int tiles_n, int *out) {
    const product::Place p = product::few_place(block, tiles_m, tiles_n);
    out[0] = p.m, out[1] = p.n;
}
int product_first_tile(int block, int grid) {
    return product::first_tile(block, grid);
}
}
