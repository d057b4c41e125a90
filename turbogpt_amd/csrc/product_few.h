// The products of product_tile.h where tiles of 128 would leave most of the GPU without work: few rows (a single token's product reads every
// weight for it) and small results.
//
// A block has 16 MT rows and 16 NT columns of the result (gated: of both matrices), and its eight waves share out k: wave w takes stages
// w, w + 8, ...  Each wave has a ring of its own in LDS, so that no wave waits for another before the end.  The copies ask for whole
// lines as in product_tile.h; fragments loaded straight from memory would ask for 16 bytes of 16 rows at a time (64 rows and 32 columns, K = 4096 in
// 8 bits: 10 us a block, here 4).  The waves' sums meet in LDS and are added in the order of the waves.
#pragma once
#include "product_shape.h"

namespace product {

constexpr int FEW_WAVES = 8;

template <bool E4M3_, bool GATED_, int MT_, int NT_, int RING_> struct Few {
    static constexpr bool E4M3 = E4M3_, GATED = GATED_;
    static constexpr int MT = MT_, NT = NT_, RING = RING_, MATRICES = GATED ? 2 : 1, TILES = MT * NT * MATRICES;
    static constexpr int A_COPIES = 2 * MT, B_COPIES = 2 * NT * MATRICES, COPIES = A_COPIES + B_COPIES + (E4M3 ? 2 : 0);
    static constexpr int SCALES_AT = (A_COPIES + B_COPIES) * 1024, SLOT_BYTES = SCALES_AT + (E4M3 ? 512 : 0); // 64 floats of rows, 64 of columns
    static constexpr int RINGS = FEW_WAVES * RING * SLOT_BYTES, MEET = FEW_WAVES * TILES * 1024, LDS_BYTES = RINGS > MEET ? RINGS : MEET;
    static_assert((RING == 1 || RING == 2) && LDS_BYTES <= 163840, "few");
};

template <class T, class Epilogue> __global__ __launch_bounds__(FEW_WAVES * 64, 2) void few_kernel(Shape s, Epilogue epilogue) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place place = few_place(blockIdx.x, s.tiles_m, s.tiles_n);
    const int m0 = place.m * T::MT * 16, n0 = place.n * T::NT * 16, row = lane & 15;
    const uint32_t ring = lds_address(lds) + wave * (T::RING * T::SLOT_BYTES);
    const int chunk = (lane & 7) ^ (lane >> 3);
    uint32_t a_offset[T::A_COPIES], b_offset[2 * T::NT];
#pragma unroll
    for (int j = 0; j < T::A_COPIES; ++j) {
        const int r = j * 8 + (lane >> 3);
        a_offset[j] = uint32_t(r < s.M - m0 ? r : s.M - m0 - 1) * uint32_t(s.lda) + chunk * 16;
    }
#pragma unroll
    for (int j = 0; j < 2 * T::NT; ++j) {
        const int r = j * 8 + (lane >> 3);
        b_offset[j] = uint32_t(r < s.N - n0 ? r : s.N - n0 - 1) * uint32_t(s.ldb) + chunk * 16;
    }
    const unsigned char *a = s.a + m0 * s.lda, *b = s.b + n0 * s.ldb;
    const int64_t low_rows = s.ldb * s.N;
    const int last_chunks = (s.k_bytes - (s.stages - 1) * STAGE + 15) >> 4; // of the last stage
    const auto request = [&](int stage, int slot) {
        const uint32_t to = ring + slot * T::SLOT_BYTES;
        // behind the end of k: the stage's first chunk
        const uint32_t back = stage + 1 == s.stages && chunk >= last_chunks ? uint32_t(chunk * 16) : 0u;
#pragma unroll
        for (int x = 0; x < T::MATRICES; ++x)
#pragma unroll
            for (int j = 0; j < 2 * T::NT; ++j)
                async_copy16(to + (T::A_COPIES + x * 2 * T::NT + j) * 1024, b + x * low_rows + stage * STAGE, b_offset[j] - back);
#pragma unroll
        for (int j = 0; j < T::A_COPIES; ++j)
            async_copy16(to + j * 1024, a + stage * STAGE, a_offset[j] - back);
        if constexpr (T::E4M3) {
            const int m = m0 + lane, n = n0 + lane;
            async_copy4(to + T::SCALES_AT, s.a_scales + int64_t(stage) * s.ld_a_scales + (m < s.M ? m : s.M - 1));
            async_copy4(to + T::SCALES_AT + 256, s.b_scales + int64_t((n < s.N ? n : s.N - 1) >> 7) * s.ld_b_scales + stage);
        }
    };
    const auto fragment = [&](uint32_t at, int half) {
        return *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(at + row * STAGE + ((((lane >> 4) + half * 4) ^ (row & 7)) << 4));
    };
    f32x4 acc[T::MT][T::NT][T::MATRICES];
#pragma unroll
    for (int i = 0; i < T::MT; ++i)
#pragma unroll
        for (int j = 0; j < T::NT; ++j)
#pragma unroll
            for (int x = 0; x < T::MATRICES; ++x)
                acc[i][j][x] = f32x4{0, 0, 0, 0};
    const int count = wave < s.stages ? (s.stages - wave + FEW_WAVES - 1) / FEW_WAVES : 0; // the wave's stages
#pragma unroll
    for (int r = 0; r < T::RING; ++r)
        if (r < count)
            request(wave + r * FEW_WAVES, r);
    int slot = 0;
    for (int i = 0; i < count; ++i) {
        const int stage = wave + i * FEW_WAVES;
        if (T::RING == 2 && i + 1 < count) // the next stage has been requested since
            wait_vmcnt<T::COPIES>();
        else
            wait_vmcnt<0>();
        const uint32_t at = ring + slot * T::SLOT_BYTES;
        if (stage + 1 == s.stages && chunk >= last_chunks) { // zeros in both operands: what lies behind a row's end may be anything
#pragma unroll
            for (int j = 0; j < T::A_COPIES + T::B_COPIES; ++j)
                *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(at + j * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
        }
        u32x4 av[T::MT][2], bv[T::NT][T::MATRICES][2];
        float row_scale[T::MT], column_scale[T::NT];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int k = 0; k < T::MT; ++k)
                av[k][h] = fragment(at + k * 2048, h);
#pragma unroll
            for (int j = 0; j < T::NT; ++j)
#pragma unroll
                for (int x = 0; x < T::MATRICES; ++x)
                    bv[j][x][h] = fragment(at + T::A_COPIES * 1024 + (x * T::NT + j) * 2048, h);
        }
        if constexpr (T::E4M3) {
            const auto scale_at = [&](int index) { return *(const __attribute__((address_space(3))) float *)(uintptr_t)(at + T::SCALES_AT + index * 4); };
#pragma unroll
            for (int k = 0; k < T::MT; ++k)
                row_scale[k] = scale_at(k * 16 + row);
#pragma unroll
            for (int j = 0; j < T::NT; ++j) // 16 columns lie in one tile of 128
                column_scale[j] = scale_at(64 + j * 16);
        }
        wait_lgkmcnt0(); // the slot may be written again
        if (i + T::RING < count)
            request(stage + T::RING * FEW_WAVES, slot);
        slot = slot + 1 == T::RING ? 0 : slot + 1;
#pragma unroll
        for (int k = 0; k < T::MT; ++k)
#pragma unroll
            for (int j = 0; j < T::NT; ++j)
#pragma unroll
                for (int x = 0; x < T::MATRICES; ++x) {
                    f32x4 &sum = acc[k][j][x];
                    if constexpr (T::E4M3) {
                        const i32x8 wide_a = __builtin_bit_cast(i32x8, __builtin_shufflevector(av[k][0], av[k][1], 0, 1, 2, 3, 4, 5, 6, 7));
                        const i32x8 wide_b = __builtin_bit_cast(i32x8, __builtin_shufflevector(bv[j][x][0], bv[j][x][1], 0, 1, 2, 3, 4, 5, 6, 7));
                        const f32x4 part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide_b, wide_a, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
                        const float scale = row_scale[k] * column_scale[j];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            sum[e] = fmaf(part[e], scale, sum[e]);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, bv[j][x][h]), __builtin_bit_cast(bf16x8, av[k][h]), sum, 0, 0, 0);
                    }
                }
    }
    __syncthreads(); // every wave has read its ring, all of whose copies have landed
    f32x4 *meet = reinterpret_cast<f32x4 *>(lds); // [wave][row tile][column tile][matrix][lane]
#pragma unroll
    for (int i = 0; i < T::MT; ++i)
#pragma unroll
        for (int j = 0; j < T::NT; ++j)
#pragma unroll
            for (int x = 0; x < T::MATRICES; ++x)
                meet[(wave * T::TILES + (i * T::NT + j) * T::MATRICES + x) * 64 + lane] = acc[i][j][x];
    __syncthreads();
    // a wave finishes a 16 x 16 tile of the result: lane l has row l % 16 and columns 4 (l / 16) .. + 3
    for (int tile = wave; tile < T::MT * T::NT; tile += FEW_WAVES) {
        f32x4 sum[T::MATRICES];
#pragma unroll
        for (int x = 0; x < T::MATRICES; ++x) {
            sum[x] = meet[(tile * T::MATRICES + x) * 64 + lane];
#pragma unroll
            for (int w = 1; w < FEW_WAVES; ++w)
                sum[x] += meet[(w * T::TILES + tile * T::MATRICES + x) * 64 + lane];
        }
        const int m = m0 + tile / T::NT * 16 + row, n = n0 + tile % T::NT * 16 + (lane >> 4) * 4;
        if (m < s.M && n < s.N)
            epilogue.template finish4<T::MATRICES>(s, sum, m, n);
    }
}

// the kernel's opt-in to more than 64 KiB of LDS, once a device
template <class Kernel> void allow_lds(Kernel kernel, std::atomic<uint64_t> &configured, int bytes) {
    int device = 0;
    check_hip(hipGetDevice(&device), "product: ");
    if (device > 63 || !(configured.load(std::memory_order_acquire) >> device & 1)) {
        check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "product LDS size: ");
        if (device < 64)
            configured.fetch_or(uint64_t(1) << device, std::memory_order_release);
    }
}

template <class T, class Epilogue> void launch_few(hipStream_t stream, Shape s, const Epilogue &epilogue) {
    s.tiles_m = (s.M + T::MT * 16 - 1) / (T::MT * 16), s.tiles_n = (s.N + T::NT * 16 - 1) / (T::NT * 16);
    s.stages = (s.k_bytes + STAGE - 1) / STAGE;
    s.tiles = s.tiles_m * s.tiles_n; // at most 256, product_kernel
    static std::atomic<uint64_t> configured;
    allow_lds(few_kernel<T, Epilogue>, configured, T::LDS_BYTES);
    hipLaunchKernelGGL((few_kernel<T, Epilogue>), dim3(s.tiles), dim3(FEW_WAVES * 64), T::LDS_BYTES, stream, s, epilogue);
    check_hip(hipGetLastError(), "product launch: ");
}

} // namespace product
