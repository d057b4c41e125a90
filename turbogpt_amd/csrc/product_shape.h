// What the products of product_tile.h and product_few.h work on.
#pragma once
#include "common.h"
#include "product_launch.h"
#include <atomic>
#include <type_traits>

namespace product {

constexpr int STAGE = 128; // bytes of k

struct Shape {
    const unsigned char *a, *b;
    int64_t lda, ldb;    // bytes from row to row
    int M, N;            // rows of a; rows of b, or (gated) half of them: columns of the result
    int k_bytes, stages; // stages = ceil(k_bytes / STAGE)
    int tiles_m, tiles_n, tiles;
    const float *a_scales, *b_scales; // of 8-bit operands: [stage][ld_a_scales] by row, [row / 128][ld_b_scales] by stage
    int ld_a_scales, ld_b_scales;
};

typedef int i32x8 __attribute__((ext_vector_type(8)));

TG_DEVICE u32x4 pack8(const float (&v)[8]) {
    return u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
}
TG_DEVICE void unpack8(const u32x4 &p, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        v[2 * e] = bf16_lo(p[e]), v[2 * e + 1] = bf16_hi(p[e]);
}
TG_DEVICE u32x2 pack4(const f32x4 &v) {
    return u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
}
TG_DEVICE f32x4 unpack4(const u32x2 &p) {
    return f32x4{bf16_lo(p.x), bf16_hi(p.x), bf16_lo(p.y), bf16_hi(p.y)};
}

} // namespace product
