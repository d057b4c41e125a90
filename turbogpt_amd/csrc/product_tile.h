// Products C[m][n] = sum_k A(m,k) B(n,k) of any number of rows and columns, for the operators whose results leave in a
// form of their own (gated.hip, gemm_q8.hip).  Both operands are k-contiguous; a row's K is `k_bytes` long, a multiple of 16.
//
// A stage is 128 bytes of k of every row of a tile, 64 values in bfloat16 and 128 in e4m3, so that every copy asks for whole
// lines and one body serves both.  Copies go straight to LDS (async_copy16).  Row r's 16-byte chunk c lies at chunk c ^ (r & 7).
// A lane's fragment of rows r0 + lane % 16 is the chunk pair lane / 16 and lane / 16 + 4: which k a chunk holds does not
// matter as long as both operands are read alike.
//
// Rows outside the operands are read as the last row inside (their results are not stored), so no address leaves the
// operands; chunks behind the end of k are read from the stage's first chunk and overwritten with zeros in both operands
// before the stage is published, as what lies behind a row's end may be anything, NaN included.
#pragma once
#include "product_few.h"

namespace product {

// WM x WN waves of (BM / WM) x 64 outputs.  AR and BR: slots of A's and B's rings; a stage is requested one less than that ahead.
// GATED: B's rows are of two matrices on top of each other, N rows each; every wave's 64 are 32 of the upper and the same 32 of the lower, and a
// tile has BN / 2 columns of the result.
//
// PHASED (256 x 256, eight waves, two on each SIMD, one of either half of the rows): a stage is cut into phases, in which a wave first reads its
// fragments and requests copies and then multiplies, and the second half of the waves is one barrier behind the first, so that on every SIMD one wave
// multiplies while the other reads.  Gated, 16384 rows, D = 768, F = 2048, pre-activations kept: tiles of 128 x 128 without phases 164 us, these 113 to 120; the
// same tiles without phases 134 (8-bit ones do not keep their sums in registers so).  In bfloat16 two phases a stage, by halves of k (four: 5 %
// slower), and three slots for A; in 8 bits four phases, by rows, as a matrix instruction takes the whole block of k.
// What bounds them: bfloat16 runs at 1.8 to 1.9 GHz with the matrix pipe busy 65 to 70 % of the cycles (8192 k), 1.6 us a stage with every unit at work; copies alone take
// 1.1, all but the copies 1.2.  8 bits, at 2.1 GHz: 2.1 us; without scaling the products 1.8, without copies 1.55, without products 1.6, without
// scaling and copies 1.2, so no one thing bounds it.  Tried there, all within 3 %: two phases; copies spread otherwise; both operands two stages ahead, into the
// half of a slot that its phase has left; scaling put off to the next phase; no phases, one barrier a stage, fragments a row ahead.  Instructions of
// 32 x 32 results: 5 to 8 % slower.  In bfloat16: three slots for
// A or two, copies before or behind the reads, both operands in the first phase, units started in turn so that their epilogues do not meet: nothing or slower.
template <bool E4M3_, bool GATED_, int BM_, int BN_, int WM_, int WN_, int AR_, bool PHASED_ = false> struct Tile {
    static constexpr int BR = PHASED_ ? 2 : AR_;
    static constexpr bool E4M3 = E4M3_, GATED = GATED_, PHASED = PHASED_;
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, AR = AR_, WAVES = WM * WN, THREADS = WAVES * 64;
    static constexpr int FM = BM / WM / 16, FN = 4, COLUMNS = GATED ? BN / 2 : BN;
    static constexpr int A_COPIES = BM / 8 / WAVES, B_COPIES = BN / 8 / WAVES, SCALE_COPIES = E4M3 ? 1 : 0;
    static constexpr int A_BYTES = BM * STAGE, B_BYTES = BN * STAGE;
    static constexpr int SCALE_BYTES = E4M3 ? BM * 4 + 256 : 0; // a slot: the rows' scales, then 64 floats of the columns'
    static constexpr int STAGING_BYTES = 4096;                  // a wave's 16 x 64 results
    static constexpr int B_AT = AR * A_BYTES, SCALES_AT = B_AT + BR * B_BYTES, LDS_BYTES = SCALES_AT + AR * SCALE_BYTES;
    static_assert(BN / WN == 64 && BN <= 256 && BM / 64 <= WAVES / (E4M3 ? 2 : 1) && B_BYTES >= WAVES * STAGING_BYTES, "tile");
};

// the wave's 16 x 64 results of fragment row i, left in its staging buffer: 16-byte chunk c (4 columns) of row r at c ^ r
template <class T> TG_DEVICE void stage_results(const f32x4 (&row)[T::FN], unsigned char *staging, int lane) {
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
        *reinterpret_cast<f32x4 *>(staging + r * 256 + (((j * 4 + g) ^ r) << 4)) = row[j];
}
// columns 8 q .. 8 q + 7 of row r of them
TG_DEVICE void staged8(const unsigned char *staging, int r, int q, float (&v)[8]) {
    const f32x4 lo = *reinterpret_cast<const f32x4 *>(staging + r * 256 + (((2 * q) ^ r) << 4));
    const f32x4 hi = *reinterpret_cast<const f32x4 *>(staging + r * 256 + (((2 * q + 1) ^ r) << 4));
#pragma unroll
    for (int e = 0; e < 4; ++e)
        v[e] = lo[e], v[4 + e] = hi[e];
}
// Tiles are walked in bands of four rows of tiles, column by column: 32 neighbours, what an XCD works on at a time, are 4 x 8 tiles
// and share 12 panels of the operands in its L2, where 32 in one row would share 33.
constexpr int BAND = 4;
TG_DEVICE void place(const Shape &s, int tile, int &tm, int &tn) {
    const int per_band = BAND * s.tiles_n, band = tile / per_band, in = tile - band * per_band;
    const int rows = s.tiles_m - band * BAND < BAND ? s.tiles_m - band * BAND : BAND;
    tn = in / rows;
    tm = band * BAND + in - tn * rows;
}

// One operand's place in the block's list of stages, and the lane's addresses there.
template <class T, bool IS_A> struct Producer {
    static constexpr int COPIES = IS_A ? T::A_COPIES : T::B_COPIES;
    int tile, stage, slot;
    const unsigned char *base; // the tile's first row
    uint32_t offset[COPIES];   // of the lane's row and chunk
    int64_t low_rows;          // bytes from the upper matrix's rows to the lower one's
    int m0, n0;                // the tile's first row; its column in tiles

    TG_DEVICE void start(const Shape &s, int first_tile, int wave, int lane) {
        tile = first_tile, stage = 0, slot = 0;
        low_rows = s.ldb * s.N;
        enter(s, wave, lane);
    }
    TG_DEVICE void enter(const Shape &s, int wave, int lane) {
        int tm, tn;
        place(s, tile, tm, tn);
        const int first = IS_A ? tm * T::BM : tn * T::COLUMNS, rows = IS_A ? s.M : s.N;
        const int64_t ld = IS_A ? s.lda : s.ldb;
        base = (IS_A ? s.a : s.b) + first * ld;
        m0 = tm * T::BM, n0 = tn;
        const int chunk = (lane & 7) ^ (lane >> 3);
#pragma unroll
        for (int j = 0; j < COPIES; ++j) {
            const int group = j * T::WAVES + wave; // of 8 rows
            int row = group * 8 + (lane >> 3);
            if (T::GATED && !IS_A)
                row = (group >> 3) * 32 + (group & 3) * 8 + (lane >> 3);
            row = row < rows - first ? row : rows - first - 1;
            offset[j] = uint32_t(row) * uint32_t(ld) + chunk * 16;
        }
    }
    // chunks of this stage that the operands have
    TG_DEVICE int chunks(const Shape &s) const { return (s.k_bytes - stage * STAGE + 15) >> 4; }
    TG_DEVICE void copy(const Shape &s, uint32_t ring, int wave, int lane) const {
        const int chunk = (lane & 7) ^ (lane >> 3), have = chunks(s);
        const uint32_t back = chunk < have ? 0u : uint32_t(chunk * 16); // behind the end of k: the stage's first chunk
        const uint32_t to = ring + slot * (IS_A ? T::A_BYTES : T::B_BYTES);
#pragma unroll
        for (int j = 0; j < COPIES; ++j) {
            const int group = j * T::WAVES + wave;
            const unsigned char *from = base + stage * STAGE;
            if (T::GATED && !IS_A && (group & 4))
                from += low_rows;
            async_copy16(to + group * 1024, from, offset[j] - back);
        }
    }
    // A's rows' scales by one half of the waves, the columns' by the other: 64 floats each
    TG_DEVICE void copy_scales(const Shape &s, uint32_t ring, int wave, int lane) const {
        const uint32_t to = ring + slot * T::SCALE_BYTES;
        if (wave < T::WAVES / 2) {
            const int part = wave % (T::BM / 64), m = m0 + part * 64 + lane;
            async_copy4(to + part * 256, s.a_scales + int64_t(stage) * s.ld_a_scales + (m < s.M ? m : s.M - 1));
        } else {
            const int first = n0 * (T::BN / 128), last = (s.N - 1) / 128;
            const int n = first + (lane & 1) < last ? first + (lane & 1) : last;
            async_copy4(to + T::BM * 4, s.b_scales + int64_t(n) * s.ld_b_scales + stage);
        }
    }
    // after the wave's copies of a stage with too few chunks have landed, where they lie in `slot_at`
    TG_DEVICE static void clear_tail(uint32_t slot_at, int have, int wave, int lane) {
        const int chunk = (lane & 7) ^ (lane >> 3);
        if (chunk < have)
            return;
#pragma unroll
        for (int j = 0; j < COPIES; ++j)
            *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(slot_at + (j * T::WAVES + wave) * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
    }
    TG_DEVICE void advance(const Shape &s, int step, int wave, int lane) {
        slot = slot + 1 == (IS_A ? T::AR : T::BR) ? 0 : slot + 1;
        if (stage + 1 < s.stages)
            ++stage;
        else if (tile + step < s.tiles) // otherwise the last stage again: the number of copies in flight stays the same
            tile += step, stage = 0, enter(s, wave, lane);
    }
};

// The value is there by now: products whose results are used phases later would otherwise be moved behind the barriers.
TG_DEVICE void pin(f32x4 &v) {
    asm volatile("" : "+v"(v));
}

template <class T, class Epilogue> __global__ __launch_bounds__(T::THREADS, T::LDS_BYTES > 81920 ? T::WAVES / 4 : T::WAVES / 2)
void tile_kernel(Shape s, Epilogue epilogue) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / T::WN, wn = wave % T::WN, step = gridDim.x;
    const uint32_t at = lds_address(lds);
    Producer<T, true> pa;
    Producer<T, false> pb;
    pa.start(s, first_tile(blockIdx.x, step), wave, lane);
    pb.start(s, first_tile(blockIdx.x, step), wave, lane);
    const auto request_a = [&] {
        if constexpr (T::E4M3)
            pa.copy_scales(s, at + T::SCALES_AT, wave, lane);
        pa.copy(s, at, wave, lane);
        pa.advance(s, step, wave, lane);
    };
    const auto request_b = [&] {
        pb.copy(s, at + T::B_AT, wave, lane);
        pb.advance(s, step, wave, lane);
    };
    request_b();
    request_a();
#pragma unroll
    for (int ahead = 2; ahead < T::AR; ++ahead) {
        if (!T::PHASED)
            request_b();
        request_a();
    }
    const int tail = (s.k_bytes % STAGE + 15) >> 4; // chunks of the last stage, 0: all
    // The wave's copies of the next stage are there.  In phases the first half of the waves asks behind its last products, the second in front of them: that
    // is the same turn, the one before the first half reads that stage.
    const auto landed = [&](bool is_tail, int slot_a, int slot_b) {
        wait_vmcnt<(T::AR - 2) * (T::A_COPIES + T::SCALE_COPIES + (T::PHASED ? 0 : T::B_COPIES))>();
        if (is_tail) {
            Producer<T, true>::clear_tail(at + slot_a * T::A_BYTES, tail, wave, lane);
            Producer<T, false>::clear_tail(at + T::B_AT + slot_b * T::B_BYTES, tail, wave, lane);
            wait_lgkmcnt0();
        }
    };
    // behind it, what the wave has read from LDS may be overwritten
    const auto turn = [] {
        __builtin_amdgcn_sched_barrier(0);
        wait_lgkmcnt0();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto publish = [&](bool is_tail, int slot_a, int slot_b) {
        landed(is_tail, slot_a, slot_b);
        turn();
    };
    publish(tail && s.stages == 1, 0, 0);
    int slot_a = 0, slot_b = 0;
    const uint32_t lane_at = (lane & 15) * STAGE + (((lane >> 4) ^ (lane & 7)) << 4);
    const auto block_at = [](uint32_t address) { // both chunks of a lane
        const u32x4 low = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)address, high = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(address ^ 64);
        return __builtin_bit_cast(i32x8, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    const auto chunk_at = [](uint32_t address) { return *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)address; };
    for (int tile = first_tile(blockIdx.x, step); tile < s.tiles; tile += step) {
        f32x4 acc[T::FM][T::FN];
#pragma unroll
        for (int i = 0; i < T::FM; ++i)
#pragma unroll
            for (int j = 0; j < T::FN; ++j)
                acc[i][j] = f32x4{0, 0, 0, 0};
        constexpr int PHASES = 4, ROWS = T::FM / PHASES ? T::FM / PHASES : 1; // 8-bit: phases, and fragment rows of each
        if (T::PHASED && wm == 1)
            turn(); // from here to the end of the tile one turn behind the other half
        for (int stage = 0; stage < s.stages; ++stage) {
            const uint32_t a_at = at + slot_a * T::A_BYTES + wm * (T::FM * 16 * STAGE) + lane_at;
            const uint32_t b_at = at + T::B_AT + slot_b * T::B_BYTES + wn * (T::FN * 16 * STAGE) + lane_at;
            const unsigned char *scales = lds + T::SCALES_AT + slot_a * T::SCALE_BYTES;
            const int next = stage + 1 < s.stages ? stage + 1 : 0; // of this tile or the block's next
            const bool next_is_tail = tail && next + 1 == s.stages;
            const int next_a = slot_a + 1 == T::AR ? 0 : slot_a + 1, next_b = slot_b + 1 == T::BR ? 0 : slot_b + 1;
            if constexpr (T::PHASED) {
                if constexpr (T::E4M3) {
                    i32x8 b[T::FN];
                    float column;
#pragma unroll
                    for (int phase = 0; phase < PHASES; ++phase) {
                        if (phase == 0) {
                            column = *reinterpret_cast<const float *>(scales + T::BM * 4 + ((wn * 64) >> 7) * 4);
#pragma unroll
                            for (int j = 0; j < T::FN; ++j)
                                b[j] = block_at(b_at + j * 2048);
                        }
                        i32x8 a[ROWS];
                        float scale[ROWS];
#pragma unroll
                        for (int i = 0; i < ROWS; ++i) {
                            const int row = phase * ROWS + i;
                            a[i] = block_at(a_at + row * 2048);
                            scale[i] = *reinterpret_cast<const float *>(scales + (wm * T::FM * 16 + row * 16 + (lane & 15)) * 4);
                        }
                        if (phase == 0)
                            request_b();
                        if (phase == 1)
                            request_a();
                        if (phase == PHASES - 1 && wm == 1)
                            landed(next_is_tail, next_a, next_b);
                        turn();
#pragma unroll
                        for (int i = 0; i < ROWS; ++i)
                            scale[i] *= column;
                        __builtin_amdgcn_s_setprio(1);
                        // a product is scaled and added two products later: one product's time is less than the matrix pipe's latency
                        f32x4 part[3];
#pragma unroll
                        for (int n = 0; n < ROWS * T::FN + 2; ++n) {
                            if (n < ROWS * T::FN)
                                part[n % 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[n % T::FN], a[n / T::FN], f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
                            __builtin_amdgcn_sched_barrier(0);
                            if (n >= 2) {
                                const int d = n - 2;
                                f32x4 &sum = acc[phase * ROWS + d / T::FN][d % T::FN];
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    sum[e] = fmaf(part[d % 3][e], scale[d / T::FN], sum[e]);
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
#pragma unroll
                        for (int n = 0; n < ROWS * T::FN; ++n)
                            pin(acc[phase * ROWS + n / T::FN][n % T::FN]);
                        __builtin_amdgcn_s_setprio(0);
                        if (phase == PHASES - 1 && wm == 0)
                            landed(next_is_tail, next_a, next_b);
                        turn();
                    }
                } else {
#pragma unroll
                    for (int phase = 0; phase < 2; ++phase) {
                        const int flip = phase * 64;
                        bf16x8 a[T::FM], b[T::FN];
#pragma unroll
                        for (int j = 0; j < T::FN; ++j)
                            b[j] = __builtin_bit_cast(bf16x8, chunk_at((b_at + j * 2048) ^ flip));
#pragma unroll
                        for (int i = 0; i < T::FM; ++i)
                            a[i] = __builtin_bit_cast(bf16x8, chunk_at((a_at + i * 2048) ^ flip));
                        if (phase == 0)
                            request_b();
                        else {
                            request_a();
                            if (wm == 1)
                                landed(next_is_tail, next_a, next_b);
                        }
                        turn();
                        __builtin_amdgcn_s_setprio(1);
#pragma unroll
                        for (int i = 0; i < T::FM; ++i)
#pragma unroll
                            for (int j = 0; j < T::FN; ++j)
                                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < T::FM; ++i)
#pragma unroll
                            for (int j = 0; j < T::FN; ++j)
                                pin(acc[i][j]);
                        __builtin_amdgcn_s_setprio(0);
                        if (phase == 1 && wm == 0)
                            landed(next_is_tail, next_a, next_b);
                        turn();
                    }
                }
            } else {
                request_b();
                request_a();
                u32x4 b[T::FN][2];
#pragma unroll
                for (int j = 0; j < T::FN; ++j) {
                    b[j][0] = chunk_at(b_at + j * 2048);
                    b[j][1] = chunk_at((b_at + j * 2048) ^ 64);
                }
                if constexpr (T::E4M3) {
                    const float column = *reinterpret_cast<const float *>(scales + T::BM * 4 + ((wn * 64) >> 7) * 4);
#pragma unroll
                    for (int i = 0; i < T::FM; ++i) {
                        const float scale = column * *reinterpret_cast<const float *>(scales + (wm * T::FM * 16 + i * 16 + (lane & 15)) * 4);
                        const i32x8 a = block_at(a_at + i * 2048);
#pragma unroll
                        for (int j = 0; j < T::FN; ++j) {
                            const i32x8 w = __builtin_bit_cast(i32x8, __builtin_shufflevector(b[j][0], b[j][1], 0, 1, 2, 3, 4, 5, 6, 7));
                            const f32x4 part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                acc[i][j][e] = fmaf(part[e], scale, acc[i][j][e]);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < T::FM; ++i) {
                        const bf16x8 low = __builtin_bit_cast(bf16x8, chunk_at(a_at + i * 2048));
                        const bf16x8 high = __builtin_bit_cast(bf16x8, chunk_at((a_at + i * 2048) ^ 64));
#pragma unroll
                        for (int j = 0; j < T::FN; ++j) {
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b[j][0]), low, acc[i][j], 0, 0, 0);
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b[j][1]), high, acc[i][j], 0, 0, 0);
                        }
                    }
                }
            }
            slot_a = next_a, slot_b = next_b;
            if constexpr (!T::PHASED)
                publish(next_is_tail, slot_a, slot_b);
        }
        if (T::PHASED && wm == 0)
            turn();
        // every wave has left B's slot that was read last, and no copy into it has been requested yet
        int tm, tn;
        place(s, tile, tm, tn);
        const int m_base = tm * T::BM + wm * T::FM * 16, n_base = tn * T::COLUMNS + wn * (T::COLUMNS / T::WN);
        unsigned char *staging = lds + T::B_AT + (slot_b ? slot_b - 1 : T::BR - 1) * T::B_BYTES + wave * T::STAGING_BYTES;
        // Without a branch where the wave's results are all inside: behind one, how many stores are in flight is not known, and every load would be
        // awaited together with the stores before it.
        if (m_base + T::FM * 16 <= s.M && n_base + T::COLUMNS / T::WN <= s.N)
            epilogue.template finish<T, true>(s, acc, staging, m_base, n_base, lane);
        else
            epilogue.template finish<T, false>(s, acc, staging, m_base, n_base, lane);
        wait_lgkmcnt0();
        turn(); // the next stage's copies go into that slot
    }
    wait_vmcnt<0>(); // no copy may land after the block's LDS has gone to another
}

// A lane's offset into a tile is 32 bits wide: 256 rows of at most 2^22 bytes.
constexpr int MOST_LD = 1 << 21;   // elements of 16 bits
constexpr int MOST_ROWS = 1 << 30; // of either operand

template <class T, class Epilogue> void launch_tiles(hipStream_t stream, Shape s, const Epilogue &epilogue) {
    s.tiles_m = (s.M + T::BM - 1) / T::BM, s.tiles_n = (s.N + T::COLUMNS - 1) / T::COLUMNS;
    require(int64_t(s.tiles_m) * s.tiles_n < (int64_t(1) << 30), "product: too many tiles");
    s.tiles = s.tiles_m * s.tiles_n, s.stages = (s.k_bytes + STAGE - 1) / STAGE;
    constexpr int most = most_blocks(T::BM == 256 ? TILES_256 : TILES_128);
    static_assert(most == (T::LDS_BYTES > 81920 ? 256 : 512), "tiles: blocks of a unit");
    static std::atomic<uint64_t> configured;
    allow_lds(tile_kernel<T, Epilogue>, configured, T::LDS_BYTES);
    hipLaunchKernelGGL((tile_kernel<T, Epilogue>), dim3(s.tiles < most ? s.tiles : most), dim3(T::THREADS), T::LDS_BYTES, stream, s, epilogue);
    check_hip(hipGetLastError(), "product launch: ");
}
template <bool E4M3, bool GATED, class Epilogue> void launch_product(hipStream_t stream, Shape s, const Epilogue &epilogue) {
    switch (product_kernel(s.M, s.N, (s.k_bytes + STAGE - 1) / STAGE, E4M3, GATED)) {
    case FEW_16:
        return launch_few<Few<E4M3, GATED, 1, 1, 2>>(stream, s, epilogue);
    case FEW_32:
        return launch_few<Few<E4M3, GATED, 2, 2, 1>>(stream, s, epilogue);
    case FEW_64x32:
        return launch_few<Few<E4M3, GATED, 4, 2, 1>>(stream, s, epilogue);
    case FEW_64:
        if constexpr (!GATED)
            return launch_few<Few<E4M3, GATED, 4, 4, 1>>(stream, s, epilogue);
        break;
    case TILES_64x128:
        return launch_tiles<Tile<E4M3, GATED, 64, 128, 2, 2, 3>>(stream, s, epilogue);
    case TILES_128:
        return launch_tiles<Tile<E4M3, GATED, 128, 128, 2, 2, 2>>(stream, s, epilogue);
    case TILES_256:
        return launch_tiles<Tile<E4M3, GATED, 256, 256, 2, 4, E4M3 ? 2 : 3, true>>(stream, s, epilogue);
    }
}

} // namespace product
