// RMS norm with the residual's addition, output in bfloat16 and / or e4m3 with a scale for each row and 128 columns, its
// backward pass, and the quantisers of rows and of weights.  The reference's norm (normalize and norm_backward,
// cuda/ops.cuh:57-80) at any width.
//
//   h = RN_bf16(x + residual), s = 1 / sqrt(mean(h^2) + eps), v = h s gamma; y = RN_bf16(v)
//   scale = max(max |v| over the row's 128 columns / 448, 2^-100), q = RN_e4m3(v / scale)
//   dx = RN(residual gradient + s gamma dy - h s^3 mean(h gamma dy)), dgamma = sum over rows of dy h s
//
// All of them are bound by memory: a row is read once, held in registers while its sum of squares is taken, and written.
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
// RN_e4m3(v / scale): a true quotient, so that codes are those of the definition; |v / scale| <= 448 (1 + 2^-23), which rounds to 448
TG_DEVICE u32x2 encode8(const float (&v)[8], float scale) {
    u32x2 code;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * e] / scale, v[4 * e + 1] / scale, 0, false);
        code[e] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * e + 2] / scale, v[4 * e + 3] / scale, word, true));
    }
    return code;
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

template <int NC, int WAVES>
__global__ __launch_bounds__(256) void rmsnorm_fwd_kernel(const bf16_t *x, const bf16_t *residual, const uint16_t *__restrict__ gamma_hi,
                                                          const uint16_t *__restrict__ gamma_lo, bf16_t *sum, bf16_t *__restrict__ y,
                                                          uint8_t *__restrict__ q, float *__restrict__ scales, int ld_scales, int rows, int D, float eps) {
    constexpr int LANES = 64 * WAVES, SLOTS = 4 / WAVES;
    __shared__ float shared[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, chunks = D >> 3;
    const float inv_d = 1.0f / D;
    for (int row0 = blockIdx.x * SLOTS; row0 < rows; row0 += gridDim.x * SLOTS) {
        const int row = row0 + slot;
        const bool live = row < rows;
        float v[NC][8];
        float squares = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = lane + j * LANES;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[j][e] = 0.f;
            if (live && c < chunks) {
                const size_t at = size_t(row) * D + c * 8;
                unpack8(*reinterpret_cast<const u32x4 *>(x + at), v[j]);
                if (residual) {
                    float add[8];
                    unpack8(*reinterpret_cast<const u32x4 *>(residual + at), add);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        v[j][e] += add[e];
                    const u32x4 h = pack8(v[j]);
                    *reinterpret_cast<u32x4 *>(sum + at) = h;
                    unpack8(h, v[j]); // the norm is of what the next operators read
                }
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    squares = fmaf(v[j][e], v[j][e], squares);
            }
        }
        const float inv = 1.0f / sqrtf(row_sum<WAVES>(squares, shared, wave) * inv_d + eps);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = lane + j * LANES;
            if (live && c < chunks) {
                float gamma[8];
                join8(*reinterpret_cast<const u32x4 *>(gamma_hi + c * 8), *reinterpret_cast<const u32x4 *>(gamma_lo + c * 8), gamma);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[j][e] = v[j][e] * inv * gamma[e];
                if (y)
                    *reinterpret_cast<u32x4 *>(y + size_t(row) * D + c * 8) = pack8(v[j]);
            }
            if (q) { // whole waves: lanes behind the last column hold zeros
                const float scale = scale_of(max_of_16(largest8(v[j])));
                if (live && c < chunks) {
                    *reinterpret_cast<u32x2 *>(q + size_t(row) * D + c * 8) = encode8(v[j], scale);
                    if ((c & 15) == 0)
                        scales[size_t(c >> 4) * ld_scales + row] = scale;
                }
            }
        }
    }
}

// dx, and a partial row of dgamma per slot into partial[block * SLOTS + slot][D]
template <int NC, int WAVES>
__global__ __launch_bounds__(256) void rmsnorm_bwd_kernel(const bf16_t *__restrict__ x, const bf16_t *__restrict__ dy, const uint16_t *__restrict__ gamma_hi,
                                                          const uint16_t *__restrict__ gamma_lo, const bf16_t *residual, bf16_t *dx,
                                                          float *__restrict__ partial, int rows, int D, float eps) {
    constexpr int LANES = 64 * WAVES, SLOTS = 4 / WAVES;
    __shared__ float shared[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, chunks = D >> 3;
    const float inv_d = 1.0f / D;
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
    for (int row0 = blockIdx.x * SLOTS; row0 < rows; row0 += gridDim.x * SLOTS) {
        const int row = row0 + slot;
        const bool live = row < rows;
        float h[NC][8], t[NC][8];
        float squares = 0.f, dot = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = lane + j * LANES;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                h[j][e] = t[j][e] = 0.f;
            if (live && c < chunks) {
                unpack8(*reinterpret_cast<const u32x4 *>(x + size_t(row) * D + c * 8), h[j]);
                unpack8(*reinterpret_cast<const u32x4 *>(dy + size_t(row) * D + c * 8), t[j]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                squares = fmaf(h[j][e], h[j][e], squares);
                dot = fmaf(h[j][e], gamma[j][e] * t[j][e], dot);
            }
        }
        const float inv = 1.0f / sqrtf(row_sum<WAVES>(squares, shared, wave) * inv_d + eps);
        const float pull = row_sum<WAVES>(dot, shared, wave) * inv_d * inv * inv; // of h, relative to gamma dy
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = lane + j * LANES;
            if (live && c < chunks) {
                const size_t at = size_t(row) * D + c * 8;
                float d[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    d[e] = inv * (gamma[j][e] * t[j][e] - h[j][e] * pull);
                    dgamma[j][e] = fmaf(t[j][e], h[j][e] * inv, dgamma[j][e]);
                }
                if (residual) { // added in 32 bits and rounded once
                    float add[8];
                    unpack8(*reinterpret_cast<const u32x4 *>(residual + at), add);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        d[e] += add[e];
                }
                *reinterpret_cast<u32x4 *>(dx + at) = pack8(d);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int c = lane + j * LANES;
        if (c < chunks) {
            float *to = partial + size_t(blockIdx.x * SLOTS + slot) * D + c * 8;
            *reinterpret_cast<f32x4 *>(to) = f32x4{dgamma[j][0], dgamma[j][1], dgamma[j][2], dgamma[j][3]};
            *reinterpret_cast<f32x4 *>(to + 4) = f32x4{dgamma[j][4], dgamma[j][5], dgamma[j][6], dgamma[j][7]};
        }
    }
}

// the partial rows' sum in a fixed order: sixteen phases, each of every sixteenth row
__global__ __launch_bounds__(256) void rmsnorm_bwd_reduce_kernel(const float *__restrict__ partial, int count, int D, float *__restrict__ dgamma, int accumulate) {
    __shared__ float part[16][17];
    const int col = threadIdx.x & 15, phase = threadIdx.x >> 4, i = blockIdx.x * 16 + col;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < D)
        for (int b = phase; b < count; b += 64)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (b + 16 * u < count)
                    s[u] += partial[size_t(b + 16 * u) * D + i];
    part[phase][col] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (phase == 0 && i < D) {
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < 16; ++p)
            sum += part[p][col];
        dgamma[i] = accumulate ? dgamma[i] + sum : sum;
    }
}

// a lane takes 8 columns, 16 lanes a group; a wave 512 columns of a row
__global__ __launch_bounds__(256) void quantize_rows_kernel(const bf16_t *__restrict__ x, int ldx, uint8_t *__restrict__ q, int ldq, float *__restrict__ scales,
                                                            int ld_scales, int rows, int columns, int parts) {
    const int lane = threadIdx.x & 63;
    const int64_t items = int64_t(rows) * parts;
    for (int64_t item = blockIdx.x * 4 + (threadIdx.x >> 6); item < items; item += gridDim.x * 4) {
        const int row = int(item / parts), c = (int(item % parts) * 64 + lane) * 8;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (c < columns)
            unpack8(*reinterpret_cast<const u32x4 *>(x + size_t(row) * ldx + c), v);
        const float scale = scale_of(max_of_16(largest8(v)));
        if (c < columns) {
            *reinterpret_cast<u32x2 *>(q + size_t(row) * ldq + c) = encode8(v, scale);
            if ((lane & 15) == 0)
                scales[size_t(c >> 7) * ld_scales + row] = scale;
        }
    }
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

constexpr int MOST_D = 8192;
void pointer(const void *p, int alignment, const char *what) {
    if (!p || reinterpret_cast<uintptr_t>(p) & (alignment - 1))
        throw std::invalid_argument(std::string(what) + ": must be non-null and " + std::to_string(alignment) + "-byte aligned");
}
void norm_shape(int rows, int D, float eps, const char *where) {
    if (rows < 1 || D < 8 || D % 8 || D > MOST_D || !(eps >= 0.f) || std::isinf(eps))
        throw std::invalid_argument(std::string(where) + ": rows at least 1, D a multiple of 8 and at most 8192, eps finite and not negative");
}
int slots_of(int D) { return D <= 2048 ? 4 : 1; } // rows a block works on at a time
int forward_blocks(int rows, int D) {
    const int need = (rows + slots_of(D) - 1) / slots_of(D);
    return need < 2048 ? need : 2048;
}
int backward_blocks(int rows, int D) {
    const int need = (rows + 2 * slots_of(D) - 1) / (2 * slots_of(D));
    return need < 768 ? need : 768;
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
            hipLaunchKernelGGL((rmsnorm_fwd_kernel<nc(), waves()>), dim3(forward_blocks(rows, D)), dim3(256), 0, stream, x, residual, gamma_hi, gamma_lo, sum, y, q,
                               scales, ld_scales, rows, D, eps);
        });
        check_hip(hipGetLastError(), "rmsnorm_fwd launch: ");
    });
}

extern "C" size_t tgk_rmsnorm_bwd_workspace(int rows, int D) {
    return rows > 0 && D > 0 && D <= MOST_D ? size_t(backward_blocks(rows, D)) * slots_of(D) * D * sizeof(float) : 0;
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
            hipLaunchKernelGGL((rmsnorm_bwd_kernel<nc(), waves()>), dim3(blocks), dim3(256), 0, stream, x, dy, gamma_hi, gamma_lo, residual, dx, partial, rows, D, eps);
        });
        hipLaunchKernelGGL(rmsnorm_bwd_reduce_kernel, dim3((D + 15) / 16), dim3(256), 0, stream, partial, blocks * slots_of(D), D, dgamma, accumulate);
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
        const int parts = (columns + 511) / 512;
        const int64_t need = (int64_t(rows) * parts + 3) / 4;
        hipLaunchKernelGGL(quantize_rows_kernel, dim3(need < 4096 ? int(need) : 4096), dim3(256), 0, stream, x, ldx, q, ldq, scales, ld_scales, rows, columns, parts);
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
        require(int64_t(tiles_m) * tiles_n < (int64_t(1) << 30), "quantize_tiles: too many tiles");
        hipLaunchKernelGGL(quantize_tiles_kernel, dim3(tiles_m * tiles_n), dim3(256), 0, stream, w, ldw, q, ldq, scales, ld_scales, rows, columns, tiles_n);
        check_hip(hipGetLastError(), "quantize_tiles launch: ");
    });
}
