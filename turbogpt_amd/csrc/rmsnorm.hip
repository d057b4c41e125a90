// RMS norm with the residual's addition, output in bfloat16 and / or e4m3 with a scale for each row and 128 columns, its
// backward pass, and the quantisers of rows and of weights.  The reference's norm (normalize and norm_backward,
// cuda/ops.cuh:57-80) at any width.
//
//   h = RN_bf16(x + residual), s = 1 / sqrt(mean(h^2) + eps), v = h s gamma; y = RN_bf16(v)
//   scale = max(max |v| over the row's 128 columns / 448, 2^-100), q = RN_e4m3(v / scale)
//   dx = RN(residual gradient + s gamma dy - h s^3 mean(h gamma dy)), dgamma = sum over rows of dy h s
//
// All of them are bound by memory: a row is read once, held in registers while its sum of squares is taken, and written, and the next row is on its way
// meanwhile.  Where a copy of 1 GiB reaches 5.0 TB/s, medians of thirty launches: 16384 x 2048 with the sum and 8-bit output 45.5 us (5.2 TB/s), without a residual
// to bfloat16 24 (5.6); 16384 x 768 forward 19.6 (5.1), backward 20.2 (5.0) + 4.6 for the fold of dgamma; 4096 x 8192 forward 44.6 (6.0), backward with the fold 67.6
// (4.0); 16384 x 4096 backward 106 (5.0).  Rows to codes 16384 x 4096 36 to 42 (4.8 to 5.6), a weight of 4096 x 4096 12.3 (4.1).  One row: 2.3 us.
#include "common.h"
#include "../../include/tgk_kernels.h"
#include <cmath>

namespace {

constexpr float LARGEST = 448.0f;                   // of e4m3
constexpr float LEAST_SCALE = 7.88860905221011805e-31f; // 2^-100: no reciprocal or quotient overflows, and a row of zeros has a scale

TG_DEVICE void unpack8(const u32x4 &p, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        v[2 * e] = bf16_lo(p[e]), v[2 * e + 1] = bf16_hi(p[e]);
}
TG_DEVICE u32x4 pack8(const float (&v)[8]) {
    return u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
}
// fp32 parameters from their halves
TG_DEVICE void join8(const u32x4 &hi, const u32x4 &lo, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = __uint_as_float(hi[e] << 16 | (lo[e] & 0xffffu));
        v[2 * e + 1] = __uint_as_float((hi[e] & 0xffff0000u) | lo[e] >> 16);
    }
}
// the largest over a row of sixteen lanes, whose 8 columns each make one group of 128
TG_DEVICE float max_of_16(float x) {
    const auto turn = [](float v, auto control) {
        return __uint_as_float(uint32_t(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(v)), decltype(control)::value, 0xF, 0xF, true)));
    };
    x = fmaxf(x, turn(x, std::integral_constant<int, 0x128>{})); // row_ror:8
    x = fmaxf(x, turn(x, std::integral_constant<int, 0x124>{})); // row_ror:4
    x = fmaxf(x, turn(x, std::integral_constant<int, 0x4E>{}));  // quad_perm [2,3,0,1]
    return fmaxf(x, turn(x, std::integral_constant<int, 0xB1>{})); // [1,0,3,2]
}
TG_DEVICE float largest8(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        m = fmaxf(m, fabsf(v[e]));
    return m;
}
TG_DEVICE float scale_of(float largest) {
    return fmaxf(largest / LARGEST, LEAST_SCALE);
}
// RN_e4m3(v / scale), of the correctly rounded quotient: v times the rounded reciprocal, put right by its own remainder (three
// instructions where a division takes ten, and a lane has eight quotients).  |v / scale| <= 448 (1 + 2^-23), which rounds to 448.
TG_DEVICE u32x2 encode8(const float (&v)[8], float scale) {
    const float inverse = 1.0f / scale;
    float quotient[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float first = v[e] * inverse;
        quotient[e] = fmaf(fmaf(-first, scale, v[e]), inverse, first);
    }
    u32x2 code;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(quotient[4 * e], quotient[4 * e + 1], 0, false);
        code[e] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(quotient[4 * e + 2], quotient[4 * e + 3], word, true));
    }
    return code;
}

// Results larger than the L2s together go past them (`past`), smaller ones stay for the next operator: 16384 x 2048 to 8 bits 50 us through them, 44
// past; 16384 x 768 forward and backward, where the backward pass reads the sum again, 43.4 and 44.4.
constexpr size_t LARGE_RESULT = size_t(32) << 20;
template <bool PAST, class V> TG_DEVICE void store(void *to, const V &v) {
    if constexpr (PAST)
        __builtin_nontemporal_store(v, reinterpret_cast<V *>(to));
    else
        *reinterpret_cast<V *>(to) = v;
}

// WAVES waves a row, NC chunks of 8 columns a lane; a block of four waves takes 4 / WAVES rows at a time.
template <int WAVES> TG_DEVICE float row_sum(float x, float *shared, int wave) {
    x = wave_sum(x);
    if constexpr (WAVES == 1)
        return x;
    __syncthreads(); // the last row's sums have been read
    if ((threadIdx.x & 63) == 0)
        shared[wave] = x;
    __syncthreads();
    return (shared[0] + shared[1]) + (shared[2] + shared[3]);
}

// A block takes `each` rows that follow each other, so that what it writes of a group's scales lies side by side.  gamma is fetched once, and
// a row's chunks while the row before is reduced.
template <int NC, int WAVES, bool ADD, bool PAST>
__global__ __launch_bounds__(256) void rmsnorm_fwd_kernel(const bf16_t *x, const bf16_t *residual, const uint16_t *__restrict__ gamma_hi,
                                                          const uint16_t *__restrict__ gamma_lo, bf16_t *sum, bf16_t *__restrict__ y,
                                                          uint8_t *__restrict__ q, float *__restrict__ scales, int ld_scales, int rows, int each, int D, float eps) {
    constexpr int LANES = 64 * WAVES, SLOTS = 4 / WAVES;
    __shared__ float shared[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, chunks = D >> 3;
    const float inv_d = 1.0f / D;
    const int first = blockIdx.x * each, last = rows - first < each ? rows : first + each;
    u32x4 raw[NC], add[NC];
    const auto fetch = [&](int row) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = lane + j * LANES;
            raw[j] = add[j] = u32x4{0, 0, 0, 0};
            if (row < last && c < chunks) {
                raw[j] = *reinterpret_cast<const u32x4 *>(x + size_t(row) * D + c * 8);
                if constexpr (ADD)
                    add[j] = *reinterpret_cast<const u32x4 *>(residual + size_t(row) * D + c * 8);
            }
        }
    };
    fetch(first + slot);
    float gamma[NC][8];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int c = lane + j * LANES;
        if (c < chunks)
            join8(*reinterpret_cast<const u32x4 *>(gamma_hi + c * 8), *reinterpret_cast<const u32x4 *>(gamma_lo + c * 8), gamma[j]);
    }
    for (int row0 = first; row0 < last; row0 += SLOTS) {
        const int row = row0 + slot;
        const bool live = row < last;
        float v[NC][8];
        float squares = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = lane + j * LANES;
            unpack8(raw[j], v[j]);
            if constexpr (ADD) {
                float other[8];
                unpack8(add[j], other);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[j][e] += other[e];
                const u32x4 h = pack8(v[j]);
                if (live && c < chunks)
                    store<PAST>(sum + size_t(row) * D + c * 8, h);
                unpack8(h, v[j]); // the norm is of what the next operators read
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                squares = fmaf(v[j][e], v[j][e], squares);
        }
        fetch(row + SLOTS); // in place of x or the residual, `sum` is written a row behind what is read
        const float inv = 1.0f / sqrtf(row_sum<WAVES>(squares, shared, wave) * inv_d + eps);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = lane + j * LANES;
            if (c < chunks) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[j][e] = v[j][e] * inv * gamma[j][e];
                if (y && live)
                    store<PAST>(y + size_t(row) * D + c * 8, pack8(v[j]));
            }
            if (q) { // whole waves: lanes behind the last column hold zeros
                const float scale = scale_of(max_of_16(largest8(v[j])));
                if (live && c < chunks) {
                    store<PAST>(q + size_t(row) * D + c * 8, encode8(v[j], scale));
                    if ((c & 15) == 0)
                        scales[size_t(c >> 4) * ld_scales + row] = scale;
                }
            }
        }
    }
}

// dx, and a partial row of dgamma per block into partial[block][D].  Everything a row needs is requested while the row before is reduced.
template <int NC, int WAVES, bool PAST>
__global__ __launch_bounds__(256) void rmsnorm_bwd_kernel(const bf16_t *__restrict__ x, const bf16_t *__restrict__ dy, const uint16_t *__restrict__ gamma_hi,
                                                          const uint16_t *__restrict__ gamma_lo, const bf16_t *residual, bf16_t *dx,
                                                          float *__restrict__ partial, int rows, int D, float eps) {
    constexpr int LANES = 64 * WAVES, SLOTS = 4 / WAVES;
    __shared__ float shared[4];
    extern __shared__ __attribute__((aligned(16))) float fold[]; // [SLOTS][D]
    const int wave = threadIdx.x >> 6, lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, chunks = D >> 3;
    const float inv_d = 1.0f / D;
    u32x4 raw_x[NC], raw_dy[NC], raw_add[NC];
    const auto fetch = [&](int row) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = lane + j * LANES;
            raw_x[j] = raw_dy[j] = raw_add[j] = u32x4{0, 0, 0, 0};
            if (row < rows && c < chunks) {
                const size_t at = size_t(row) * D + c * 8;
                raw_x[j] = *reinterpret_cast<const u32x4 *>(x + at);
                raw_dy[j] = *reinterpret_cast<const u32x4 *>(dy + at);
                if (residual) // may be dx: a row is read by the lanes that write it, before they do
                    raw_add[j] = *reinterpret_cast<const u32x4 *>(residual + at);
            }
        }
    };
    const int step = gridDim.x * SLOTS;
    fetch(blockIdx.x * SLOTS + slot);
    float gamma[NC][8], dgamma[NC][8];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int c = lane + j * LANES;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            gamma[j][e] = dgamma[j][e] = 0.f;
        if (c < chunks)
            join8(*reinterpret_cast<const u32x4 *>(gamma_hi + c * 8), *reinterpret_cast<const u32x4 *>(gamma_lo + c * 8), gamma[j]);
    }
    for (int row0 = blockIdx.x * SLOTS; row0 < rows; row0 += step) {
        const int row = row0 + slot;
        const bool live = row < rows;
        float h[NC][8], t[NC][8];
        u32x4 add[NC];
        float squares = 0.f, dot = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            unpack8(raw_x[j], h[j]);
            unpack8(raw_dy[j], t[j]);
            add[j] = raw_add[j];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                squares = fmaf(h[j][e], h[j][e], squares);
                dot = fmaf(h[j][e], gamma[j][e] * t[j][e], dot);
            }
        }
        fetch(row + step);
        const float inv = 1.0f / sqrtf(row_sum<WAVES>(squares, shared, wave) * inv_d + eps);
        const float pull = row_sum<WAVES>(dot, shared, wave) * inv_d * inv * inv; // of h, relative to gamma dy
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = lane + j * LANES;
            if (live && c < chunks) {
                float d[8], other[8];
                unpack8(add[j], other); // zeros without a residual
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // the gradient through the norm and the residual's are added in 32 bits and rounded once
                    d[e] = fmaf(inv, gamma[j][e] * t[j][e] - h[j][e] * pull, other[e]);
                    dgamma[j][e] = fmaf(t[j][e], h[j][e] * inv, dgamma[j][e]);
                }
                store<PAST>(dx + size_t(row) * D + c * 8, pack8(d));
            }
        }
    }
    // the slots' sums, one on top of the other
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int c = lane + j * LANES;
        if (c < chunks) {
            float *to = (SLOTS == 1 ? partial + size_t(blockIdx.x) * D : fold + slot * D) + c * 8;
            *reinterpret_cast<f32x4 *>(to) = f32x4{dgamma[j][0], dgamma[j][1], dgamma[j][2], dgamma[j][3]};
            *reinterpret_cast<f32x4 *>(to + 4) = f32x4{dgamma[j][4], dgamma[j][5], dgamma[j][6], dgamma[j][7]};
        }
    }
    if constexpr (SLOTS > 1) {
        __syncthreads();
        for (int c = threadIdx.x * 4; c < D; c += 1024) {
            f32x4 total = *reinterpret_cast<const f32x4 *>(fold + c);
#pragma unroll
            for (int k = 1; k < SLOTS; ++k)
                total += *reinterpret_cast<const f32x4 *>(fold + k * D + c);
            *reinterpret_cast<f32x4 *>(partial + size_t(blockIdx.x) * D + c) = total;
        }
    }
}

// the partial rows' sum in a fixed order: 32 phases, each of every 32nd row, eight of them in flight
__global__ __launch_bounds__(256) void rmsnorm_bwd_reduce_kernel(const float *__restrict__ partial, int count, int D, float *__restrict__ dgamma, int accumulate) {
    __shared__ float part[32][9];
    const int col = threadIdx.x & 7, phase = threadIdx.x >> 3, i = blockIdx.x * 8 + col; // 8 divides D
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int b = phase; b < count; b += 256) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            v[u] = b + 32 * u < count ? partial[size_t(b + 32 * u) * D + i] : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            s[u] += v[u];
    }
    part[phase][col] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (phase == 0) {
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < 32; ++p)
            sum += part[p][col];
        dgamma[i] = accumulate ? dgamma[i] + sum : sum;
    }
}

// A lane takes 8 columns, 16 lanes a group, a wave 512 columns of a row; a block 32 rows of them, four rows of a wave in flight, and writes their
// scales side by side.
constexpr int QUANTIZE_ROWS = 32;
__global__ __launch_bounds__(256) void quantize_rows_kernel(const bf16_t *__restrict__ x, int ldx, uint8_t *__restrict__ q, int ldq, float *__restrict__ scales,
                                                            int ld_scales, int rows, int columns, int parts) {
    __shared__ float shared[4][QUANTIZE_ROWS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int part = blockIdx.x % parts, first = blockIdx.x / parts * QUANTIZE_ROWS, c = (part * 64 + lane) * 8;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        u32x4 raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = first + half * 16 + i * 4 + wave;
            raw[i] = u32x4{0, 0, 0, 0};
            if (row < rows && c < columns)
                raw[i] = *reinterpret_cast<const u32x4 *>(x + size_t(row) * ldx + c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int in = half * 16 + i * 4 + wave, row = first + in;
            float v[8];
            unpack8(raw[i], v);
            const float scale = scale_of(max_of_16(largest8(v)));
            if (row < rows && c < columns)
                *reinterpret_cast<u32x2 *>(q + size_t(row) * ldq + c) = encode8(v, scale);
            if ((lane & 15) == 0)
                shared[lane >> 4][in] = scale;
        }
    }
    __syncthreads();
    const int group = threadIdx.x / QUANTIZE_ROWS, row = first + threadIdx.x % QUANTIZE_ROWS;
    if (group < 4 && part * 512 + group * 128 < columns && row < rows)
        scales[size_t(part * 4 + group) * ld_scales + row] = shared[group][threadIdx.x % QUANTIZE_ROWS];
}

// one block a tile of 128 x 128
__global__ __launch_bounds__(256) void quantize_tiles_kernel(const bf16_t *__restrict__ w, int ldw, uint8_t *__restrict__ q, int ldq, float *__restrict__ scales,
                                                             int ld_scales, int rows, int columns, int tiles_n) {
    __shared__ float shared[4];
    const int tile_row = blockIdx.x / tiles_n, tile_column = blockIdx.x % tiles_n;
    const int c = tile_column * 128 + (threadIdx.x & 15) * 8;
    float v[8][8], largest = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = tile_row * 128 + i * 16 + (threadIdx.x >> 4);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[i][e] = 0.f;
        if (row < rows && c < columns)
            unpack8(*reinterpret_cast<const u32x4 *>(w + size_t(row) * ldw + c), v[i]);
        largest = fmaxf(largest, largest8(v[i]));
    }
    largest = wave_max(largest);
    if ((threadIdx.x & 63) == 0)
        shared[threadIdx.x >> 6] = largest;
    __syncthreads();
    const float scale = scale_of(fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3])));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = tile_row * 128 + i * 16 + (threadIdx.x >> 4);
        if (row < rows && c < columns)
            *reinterpret_cast<u32x2 *>(q + size_t(row) * ldq + c) = encode8(v[i], scale);
    }
    if (threadIdx.x == 0)
        scales[size_t(tile_row) * ld_scales + tile_column] = scale;
}

constexpr int MOST_D = 8192, MOST_ROWS = 1 << 30, MOST_BLOCKS = 1 << 24; // blocks: of 256 work items, of which a launch holds fewer than 2^32
void pointer(const void *p, int alignment, const char *what) {
    if (!p || reinterpret_cast<uintptr_t>(p) & (alignment - 1))
        throw std::invalid_argument(std::string(what) + ": must be non-null and " + std::to_string(alignment) + "-byte aligned");
}
void norm_shape(int rows, int D, float eps, const char *where) {
    if (rows < 1 || rows > MOST_ROWS || D < 8 || D % 8 || D > MOST_D || !(eps >= 0.f) || std::isinf(eps))
        throw std::invalid_argument(std::string(where) + ": rows at least 1 and at most 2^30, D a multiple of 8 and at most 8192, eps finite and not negative");
}
int slots_of(int D) { return D <= 2048 ? 4 : 1; } // rows a block works on at a time
// rows a block takes in all: one round of its slots, more where that would be more than 2048 blocks (16384 x 2048 to 8 bits 53 us with 1024, 50 with 2048)
int forward_rows(int rows, int D) {
    const int slots = slots_of(D), rounds = (rows + 2048 * slots - 1) / (2048 * slots);
    return rounds * slots;
}
// two rounds of the slots at least, and at most two blocks a unit (16384 x 768, 1024, 2048: 23.6, 28.0, 58.2 us; with three 24.2, 29.2, 63.2; with four 25.9,
// 32.6, 61.5)
int backward_blocks(int rows, int D) {
    const int need = (rows + 2 * slots_of(D) - 1) / (2 * slots_of(D));
    return need < 512 ? need : 512;
}
// f(chunks a lane, waves a row)
template <class F> void by_width(int D, F &&f) {
    using std::integral_constant;
    if (D <= 512)
        f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (D <= 1024)
        f(integral_constant<int, 2>{}, integral_constant<int, 1>{});
    else if (D <= 2048)
        f(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else
        f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
}
} // namespace

extern "C" int tgk_rmsnorm_fwd(hipStream_t stream, int rows, int D, const uint16_t *x, const uint16_t *residual, const uint16_t *gamma_hi, const uint16_t *gamma_lo,
                               uint16_t *sum, uint16_t *y, uint8_t *q, float *scales, int ld_scales, float eps) {
    return guarded([&] {
        norm_shape(rows, D, eps, "rmsnorm_fwd");
        pointer(x, 16, "rmsnorm_fwd: x");
        pointer(gamma_hi, 16, "rmsnorm_fwd: gamma_hi");
        pointer(gamma_lo, 16, "rmsnorm_fwd: gamma_lo");
        if (residual) {
            pointer(residual, 16, "rmsnorm_fwd: residual");
            pointer(sum, 16, "rmsnorm_fwd: sum (of x and the residual)");
        }
        require(y || q, "rmsnorm_fwd: no output: y and q are both NULL");
        if (y)
            pointer(y, 16, "rmsnorm_fwd: y");
        if (q) {
            pointer(q, 8, "rmsnorm_fwd: q");
            pointer(scales, 4, "rmsnorm_fwd: scales");
            require(ld_scales >= rows, "rmsnorm_fwd: ld_scales must be at least the rows");
        }
        by_width(D, [&](auto nc, auto waves) {
            const int each = forward_rows(rows, D), blocks = (rows - 1) / each + 1;
            const bool past = size_t(rows) * D * 2 > LARGE_RESULT;
            const auto kernel = past ? (residual ? rmsnorm_fwd_kernel<nc(), waves(), true, true> : rmsnorm_fwd_kernel<nc(), waves(), false, true>)
                                     : (residual ? rmsnorm_fwd_kernel<nc(), waves(), true, false> : rmsnorm_fwd_kernel<nc(), waves(), false, false>);
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, x, residual, gamma_hi, gamma_lo, sum, y, q, scales, ld_scales, rows, each, D, eps);
        });
        check_hip(hipGetLastError(), "rmsnorm_fwd launch: ");
    });
}

extern "C" size_t tgk_rmsnorm_bwd_workspace(int rows, int D) {
    return rows > 0 && rows <= MOST_ROWS && D > 0 && D <= MOST_D ? size_t(backward_blocks(rows, D)) * D * sizeof(float) : 0;
}

extern "C" int tgk_rmsnorm_bwd(hipStream_t stream, int rows, int D, const uint16_t *x, const uint16_t *dy, const uint16_t *gamma_hi, const uint16_t *gamma_lo,
                               const uint16_t *residual, uint16_t *dx, float *dgamma, float eps, int accumulate, void *workspace, size_t workspace_bytes) {
    return guarded([&] {
        norm_shape(rows, D, eps, "rmsnorm_bwd");
        pointer(x, 16, "rmsnorm_bwd: x");
        pointer(dy, 16, "rmsnorm_bwd: dy");
        pointer(gamma_hi, 16, "rmsnorm_bwd: gamma_hi");
        pointer(gamma_lo, 16, "rmsnorm_bwd: gamma_lo");
        pointer(dx, 16, "rmsnorm_bwd: dx");
        pointer(dgamma, 4, "rmsnorm_bwd: dgamma");
        if (residual)
            pointer(residual, 16, "rmsnorm_bwd: residual");
        require(workspace && !(reinterpret_cast<uintptr_t>(workspace) & 15) && workspace_bytes >= tgk_rmsnorm_bwd_workspace(rows, D),
                "rmsnorm_bwd: workspace too small or not 16-byte aligned (see tgk_rmsnorm_bwd_workspace)");
        const int blocks = backward_blocks(rows, D);
        float *partial = static_cast<float *>(workspace);
        by_width(D, [&](auto nc, auto waves) {
            const auto kernel = size_t(rows) * D * 2 > LARGE_RESULT ? rmsnorm_bwd_kernel<nc(), waves(), true> : rmsnorm_bwd_kernel<nc(), waves(), false>;
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), waves() == 1 ? 4 * D * sizeof(float) : 0, stream, x, dy, gamma_hi, gamma_lo, residual, dx, partial, rows, D, eps);
        });
        hipLaunchKernelGGL(rmsnorm_bwd_reduce_kernel, dim3(D / 8), dim3(256), 0, stream, partial, blocks, D, dgamma, accumulate);
        check_hip(hipGetLastError(), "rmsnorm_bwd launch: ");
    });
}

extern "C" int tgk_quantize_rows(hipStream_t stream, int rows, int columns, const uint16_t *x, int ldx, uint8_t *q, int ldq, float *scales, int ld_scales) {
    return guarded([&] {
        require(rows > 0 && columns > 0 && columns % 8 == 0, "quantize_rows: at least one row, columns a multiple of 8");
        pointer(x, 16, "quantize_rows: x");
        pointer(q, 8, "quantize_rows: q");
        pointer(scales, 4, "quantize_rows: scales");
        require(ldx >= columns && ldx % 8 == 0 && ldq >= columns && ldq % 8 == 0, "quantize_rows: leading dimensions must be multiples of 8, at least the columns");
        require(ld_scales >= rows, "quantize_rows: ld_scales must be at least the rows");
        const int parts = (columns - 1) / 512 + 1;
        const int64_t blocks = int64_t((rows - 1) / QUANTIZE_ROWS + 1) * parts;
        require(blocks < MOST_BLOCKS, "quantize_rows: too many rows and columns: 2^24 blocks of 32 rows and 512 columns or more");
        hipLaunchKernelGGL(quantize_rows_kernel, dim3(int(blocks)), dim3(256), 0, stream, x, ldx, q, ldq, scales, ld_scales, rows, columns, parts);
        check_hip(hipGetLastError(), "quantize_rows launch: ");
    });
}

extern "C" int tgk_quantize_tiles(hipStream_t stream, int rows, int columns, const uint16_t *w, int ldw, uint8_t *q, int ldq, float *scales, int ld_scales) {
    return guarded([&] {
        require(rows > 0 && columns > 0 && columns % 8 == 0, "quantize_tiles: at least one row, columns a multiple of 8");
        pointer(w, 16, "quantize_tiles: w");
        pointer(q, 8, "quantize_tiles: q");
        pointer(scales, 4, "quantize_tiles: scales");
        require(ldw >= columns && ldw % 8 == 0 && ldq >= columns && ldq % 8 == 0, "quantize_tiles: leading dimensions must be multiples of 8, at least the columns");
        const int tiles_m = (rows - 1) / 128 + 1, tiles_n = (columns - 1) / 128 + 1;
        require(ld_scales >= tiles_n, "quantize_tiles: ld_scales must be at least the tiles of a row");
        require(int64_t(tiles_m) * tiles_n < MOST_BLOCKS, "quantize_tiles: too many tiles: 2^24 blocks of 128 x 128 or more");
        hipLaunchKernelGGL(quantize_tiles_kernel, dim3(tiles_m * tiles_n), dim3(256), 0, stream, w, ldw, q, ldq, scales, ld_scales, rows, columns, tiles_n);
        check_hip(hipGetLastError(), "quantize_tiles launch: ");
    });
}
