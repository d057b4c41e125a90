// The gated feed-forward block, H = act(X Wg^T) * (X Wu^T), and its backward pass.  W = [Wg; Wu] is packed [2F][D], the layout
// of the width-16 network's gate and up projections (model.h:27-31; swiglu_activation and swiglu_backward, cuda/ops.cuh:120-144).
//
// Forward: one product whose tiles hold 32 gate and the same 32 up columns per wave, so that a lane has both pre-activations
// of an output and nothing but H (and, for training, the pre-activations) is written.
// Backward, from the gradient of the block's output Y = H Wd^T: dH = dY Wd is a product whose epilogue reads the saved
// pre-activations and writes dG = dH u act'(g) and dU = dH act(g); dH itself never reaches memory.  dX = [dG dU] W is a plain
// product over 2F.
//
// Measured, us, least and median of thirty launches with others between them: 16384 x 768, F = 2048 forward with both pre-activations kept 106 and 125 (103 GFLOP,
// 0.23 GB of operands and results, of which 0.202 are written, as counted, and 0.201 have to be), dH's product 81 and 91 (51 GFLOP, 0.30 GB); 16384 x 1024,
// F = 4096, GELU 254 and 270, and 187 and 195 (275 and 137 GFLOP).  dH's epilogue reads and writes four values for each sum: its memory traffic alone takes
// 112 us of the 187, the products alone 100, and as every unit comes to it with the clock and the L2s shared they add up.  One token, 1024 -> 2816: 3.9,
// 11.5 MB of weights.
//
// The weights' gradients are dW = [dG dU]^T X and dWd = dY^T H: tgk_gemm_wgrad.
#include "product_tile.h"
#include "../../include/tgk_kernels.h"

namespace {
using namespace product;

// SiLU and its derivative from one exponential: s = 1 / (1 + e^-g), g s and s (1 + g (1 - s)).  A reciprocal of an
// infinite 1 + e^-g is 0, so the far negative side gives -0 and not NaN, but g = -inf gives NaN as the formula does.
struct Gate {
    float act, slope;
};
template <int ACT> TG_DEVICE float act_f(float g) {
    if constexpr (ACT == TGK_GATE_SILU)
        return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g));
    else
        return gelu_f(g);
}
template <int ACT> TG_DEVICE Gate gate_f(float g) {
    if constexpr (ACT == TGK_GATE_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g));
        return {g * s, s * fmaf(g, 1.0f - s, 1.0f)};
    } else {
        return {gelu_f(g), gelu_grad_f(g)};
    }
}

template <int ACT, bool KEEP> struct GatedForward {
    bf16_t *h, *gu;
    int ld_h, ld_gu;
    // The activation and the product are taken of the 32-bit sums and rounded once; what is kept for the backward pass is
    // rounded by itself.
    template <class T, bool INSIDE> TG_DEVICE void finish(const Shape &s, const f32x4 (&acc)[T::FM][T::FN], unsigned char *staging, int m_base, int n_base, int lane) const {
        const int r = lane >> 2, q = lane & 3, f = n_base + q * 8;
#pragma unroll
        for (int i = 0; i < T::FM; ++i) {
            __builtin_amdgcn_sched_barrier(0); // one fragment row at a time: hoisted loads would not leave the sums their registers
            stage_results<T>(acc[i], staging, lane);
            float g[8], u[8], v[8];
            staged8(staging, r, q, g);
            staged8(staging, r, 4 + q, u);
            const int m = m_base + i * 16 + r;
            if (INSIDE || (m < s.M && f < s.N)) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = act_f<ACT>(g[e]) * u[e];
                *reinterpret_cast<u32x4 *>(h + size_t(m) * ld_h + f) = pack8(v);
                if constexpr (KEEP) {
                    *reinterpret_cast<u32x4 *>(gu + size_t(m) * ld_gu + f) = pack8(g);
                    *reinterpret_cast<u32x4 *>(gu + size_t(m) * ld_gu + s.N + f) = pack8(u);
                }
            }
        }
    }
    template <int> TG_DEVICE void finish4(const Shape &s, const f32x4 (&sum)[2], int m, int n) const {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = act_f<ACT>(sum[0][e]) * sum[1][e];
        *reinterpret_cast<u32x2 *>(h + size_t(m) * ld_h + n) = pack4(v);
        if constexpr (KEEP) {
            *reinterpret_cast<u32x2 *>(gu + size_t(m) * ld_gu + n) = pack4(sum[0]);
            *reinterpret_cast<u32x2 *>(gu + size_t(m) * ld_gu + s.N + n) = pack4(sum[1]);
        }
    }
};

template <int ACT> struct GatedBackward {
    const bf16_t *gu; // may be dgu: every lane reads its values before it writes them
    bf16_t *dgu;
    int ld_gu, ld_dgu;
    // The saved pre-activations of AHEAD fragment rows are on their way while one is finished.
    template <class T, bool INSIDE> TG_DEVICE void finish(const Shape &s, const f32x4 (&acc)[T::FM][T::FN], unsigned char *staging, int m_base, int n_base, int lane) const {
        constexpr int AHEAD = T::FM < 3 ? T::FM : 3;
        const int r = lane >> 3, q = lane & 7, f = n_base + q * 8;
        u32x4 raw[AHEAD][2][2];
        const auto fetch = [&](int i) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int m = m_base + i * 16 + half * 8 + r;
                if (INSIDE || (m < s.M && f < s.N)) {
                    const bf16_t *from = gu + size_t(m) * ld_gu + f;
                    // read once and larger than the L2s, whose lines the operands need: 16384 x 4096, D = 1024 196 us through them, 184 past them
                    raw[i % AHEAD][half][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from));
                    raw[i % AHEAD][half][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from + s.N));
                }
            }
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            fetch(i);
#pragma unroll
        for (int i = 0; i < T::FM; ++i) {
            __builtin_amdgcn_sched_barrier(0); // one fragment row at a time: hoisted loads would not leave the sums their registers
            stage_results<T>(acc[i], staging, lane);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int m = m_base + i * 16 + half * 8 + r;
                float dh[8], g[8], u[8];
                staged8(staging, half * 8 + r, q, dh);
                if (INSIDE || (m < s.M && f < s.N)) {
                    unpack8(raw[i % AHEAD][half][0], g);
                    unpack8(raw[i % AHEAD][half][1], u);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const Gate gate = gate_f<ACT>(g[e]);
                        g[e] = dh[e] * u[e] * gate.slope;
                        u[e] = dh[e] * gate.act;
                    }
                    *reinterpret_cast<u32x4 *>(dgu + size_t(m) * ld_dgu + f) = pack8(g);
                    *reinterpret_cast<u32x4 *>(dgu + size_t(m) * ld_dgu + s.N + f) = pack8(u);
                }
            }
            if (i + AHEAD < T::FM)
                fetch(i + AHEAD);
        }
    }
    template <int> TG_DEVICE void finish4(const Shape &s, const f32x4 (&dh)[1], int m, int n) const {
        f32x4 g = unpack4(*reinterpret_cast<const u32x2 *>(gu + size_t(m) * ld_gu + n)), u = unpack4(*reinterpret_cast<const u32x2 *>(gu + size_t(m) * ld_gu + s.N + n));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const Gate gate = gate_f<ACT>(g[e]);
            g[e] = dh[0][e] * u[e] * gate.slope;
            u[e] = dh[0][e] * gate.act;
        }
        *reinterpret_cast<u32x2 *>(dgu + size_t(m) * ld_dgu + n) = pack4(g);
        *reinterpret_cast<u32x2 *>(dgu + size_t(m) * ld_dgu + s.N + n) = pack4(u);
    }
};

struct Plain {
    bf16_t *out;
    int ld_out;
    template <class T, bool INSIDE> TG_DEVICE void finish(const Shape &s, const f32x4 (&acc)[T::FM][T::FN], unsigned char *staging, int m_base, int n_base, int lane) const {
#pragma unroll
        for (int i = 0; i < T::FM; ++i) {
            __builtin_amdgcn_sched_barrier(0); // one fragment row at a time: hoisted loads would not leave the sums their registers
            stage_results<T>(acc[i], staging, lane);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = (lane >> 3) + half * 8, q = lane & 7, m = m_base + i * 16 + r, n = n_base + q * 8;
                float v[8];
                staged8(staging, r, q, v);
                if (INSIDE || (m < s.M && n < s.N))
                    *reinterpret_cast<u32x4 *>(out + size_t(m) * ld_out + n) = pack8(v);
            }
        }
    }
    template <int> TG_DEVICE void finish4(const Shape &, const f32x4 (&sum)[1], int m, int n) const {
        *reinterpret_cast<u32x2 *>(out + size_t(m) * ld_out + n) = pack4(sum[0]);
    }
};

template <bool GATED, class Epilogue> void product_bf16(hipStream_t stream, int M, int N, int K, const bf16_t *a, int lda, const bf16_t *b, int ldb, const Epilogue &epilogue) {
    Shape s{};
    s.a = reinterpret_cast<const unsigned char *>(a), s.b = reinterpret_cast<const unsigned char *>(b);
    s.lda = int64_t(lda) * 2, s.ldb = int64_t(ldb) * 2;
    s.M = M, s.N = N, s.k_bytes = K * 2;
    launch_product<false, GATED>(stream, s, epilogue);
}

void operand(const void *p, int ld, int columns, const char *what) {
    if (!p || reinterpret_cast<uintptr_t>(p) & 15 || ld < columns || ld % 8 || ld > MOST_LD)
        throw std::invalid_argument(std::string(what) + ": needs a 16-byte aligned pointer and a leading dimension that is a multiple of 8, at least the columns and at most 2^21");
}
void block_shape(int M, int F, int D, int activation, const char *where) {
    if (M < 1 || M > MOST_ROWS || F < 8 || D < 8 || F % 8 || D % 8 || F > MOST_LD / 2 || D > MOST_LD)
        throw std::invalid_argument(std::string(where) + ": M at least 1 and at most 2^30, F and D multiples of 8 (F at most 2^20, D at most 2^21)");
    if (activation != TGK_GATE_SILU && activation != TGK_GATE_GELU)
        throw std::invalid_argument(std::string(where) + ": activation is TGK_GATE_SILU or TGK_GATE_GELU");
}
template <class F> void by_activation(int activation, F &&f) {
    if (activation == TGK_GATE_SILU)
        f(std::integral_constant<int, TGK_GATE_SILU>{});
    else
        f(std::integral_constant<int, TGK_GATE_GELU>{});
}
} // namespace

extern "C" int tgk_gated_fwd(hipStream_t stream, int M, int F, int D, const uint16_t *X, int ldx, const uint16_t *W, int ldw, uint16_t *H, int ldh,
                             uint16_t *GU, int ldgu, int activation) {
    return guarded([&] {
        block_shape(M, F, D, activation, "gated_fwd");
        operand(X, ldx, D, "gated_fwd: X");
        operand(W, ldw, D, "gated_fwd: W");
        operand(H, ldh, F, "gated_fwd: H");
        if (GU)
            operand(GU, ldgu, 2 * F, "gated_fwd: GU");
        by_activation(activation, [&](auto act) {
            if (GU)
                product_bf16<true>(stream, M, F, D, X, ldx, W, ldw, GatedForward<act(), true>{H, GU, ldh, ldgu});
            else
                product_bf16<true>(stream, M, F, D, X, ldx, W, ldw, GatedForward<act(), false>{H, nullptr, ldh, 0});
        });
    });
}

extern "C" int tgk_gated_bwd(hipStream_t stream, int M, int F, int D, const uint16_t *dY, int lddy, const uint16_t *Wdt, int ldwdt, const uint16_t *GU, int ldgu,
                             uint16_t *dGU, int lddgu, const uint16_t *Wt, int ldwt, uint16_t *dX, int lddx, int activation) {
    return guarded([&] {
        block_shape(M, F, D, activation, "gated_bwd");
        operand(dY, lddy, D, "gated_bwd: dY");
        operand(Wdt, ldwdt, D, "gated_bwd: Wdt");
        operand(GU, ldgu, 2 * F, "gated_bwd: GU");
        operand(dGU, lddgu, 2 * F, "gated_bwd: dGU");
        require(GU != dGU || ldgu == lddgu, "gated_bwd: in place, GU and dGU have the same leading dimension");
        if (dX) {
            operand(Wt, ldwt, 2 * F, "gated_bwd: Wt");
            operand(dX, lddx, D, "gated_bwd: dX");
        }
        by_activation(activation, [&](auto act) { product_bf16<false>(stream, M, F, D, dY, lddy, Wdt, ldwdt, GatedBackward<act()>{GU, dGU, ldgu, lddgu}); });
        if (!dX)
            return;
        // A plain product: the framework's, where it takes the shape.  With the product before it, us there and here: 16384 x 1024, F = 4096 366, 390; 8192 x 1024,
        // F = 4096 208, 239; 8192 x 640, F = 2048 88, 97; 2048 x 256, F = 1024 17.4, 22.2.  Below 1024 rows the kernels here are as fast or faster (512 x 512,
        // F = 2048 18.7, 18.2).
        if (M % 128 == 0 && M >= 1024 && (D % 128 == 0 || D % 192 == 0) && F % 16 == 0) {
            if (tgk_gemm_dgrad_t(stream, M, 2 * F, D, dGU, lddgu, Wt, ldwt, dX, lddx, nullptr, 0) < 0)
                throw std::runtime_error(tg_last_error);
            return;
        }
        product_bf16<false>(stream, M, D, 2 * F, dGU, lddgu, Wt, ldwt, Plain{dX, lddx});
    });
}
