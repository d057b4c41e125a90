"""The 8-bit linear layer against its definition in 64 bits.

Tolerance, element by element: the rounding to bfloat16 is off by 2^-8 of the value, sums in 32 bits of K products (whole
blocks of 128 are summed, behind the end of K zeros) by at most (K + 128) 2^-23 of the sum of the products' magnitudes.

The matrix instruction adds the products of eight neighbouring k with each other before it adds them to a 32-bit sum, aligned to
the largest operands' exponents with 13 bits behind them: beside 448 x 448 = 1.53 x 2^17 (exponents 8 and 8) a product of 2^3 = 2^(16 - 13) is
kept and one of 2^2 is not, among the same eight; among others 2^-6 is.  The largest product is exact (4-bit by 4-bit significands),
the seven others lose less than 2^-13 of it each: together under 7 x 2^-13 < 2^-10 of the eight's largest product, and over all of
K under 2^-10 of the sum of the products' magnitudes.  Where all products are multiples of the eight's unit nothing is
lost: test_small_integers asks for equal bits."""
import pytest
import torch

from gpu_util import check, library, stream, sync

pytestmark = pytest.mark.gpu

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
HALF = 2.0 ** -8


def codes(rows, K, ld, generator):
    """Codes of every size e4m3 has, NaN codes behind the rows' ends."""
    whole = torch.full((rows, ld), 0x7f, dtype=torch.uint8)
    values = torch.randn(rows, K, generator=generator) * torch.exp(2 * torch.randn(rows, K, generator=generator))
    whole[:, :K] = values.clamp(-448, 448).to(F8).view(torch.uint8)
    return whole.cuda()


def case(M, N, K, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    blocks = -(-K // 128)
    x, w = codes(M, K, K + pad, g), codes(N, K, K + pad, g)
    x_scales = torch.full((blocks, M + pad), float("nan"))
    x_scales[:, :M] = torch.exp(2 * torch.randn(blocks, M, generator=g))
    w_scales = torch.full((-(-N // 128), blocks + pad), float("nan"))
    w_scales[:, :blocks] = torch.exp(torch.randn(-(-N // 128), blocks, generator=g))
    return x, x_scales.cuda(), w, w_scales.cuda()


def run(M, N, K, x, x_scales, w, w_scales, residual=None, out=None, ldy=None):
    ldy = ldy or N
    y = torch.full((M + 2, ldy), 7.0, dtype=BF16, device="cuda") if out is None else out
    check(library().tgk_gemm_q8(stream(), M, N, K, x.data_ptr(), x.stride(0), x_scales.data_ptr(), x_scales.stride(0), w.data_ptr(), w.stride(0),
                                w_scales.data_ptr(), w_scales.stride(0), y.data_ptr(), ldy, residual.data_ptr() if residual is not None else None,
                                residual.stride(0) if residual is not None else 0))
    sync()
    if out is None:
        assert bool((y[M:] == 7.0).all()) and bool((y[:, N:] == 7.0).all())
    return y[:M, :N]


def values(M, N, K, x, x_scales, w, w_scales):
    blocks = -(-K // 128)
    xv = x[:, :K].view(F8).double() * x_scales[:, :M].t().double().repeat_interleave(128, 1)[:, :K]
    per_tile = w_scales[:, :blocks].double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    return xv, w[:, :K].view(F8).double() * per_tile[:N, :K]


def near(got, want, bound, what):
    over = (got.double() - want).abs() - bound
    assert bool((over <= 0).all()), f"{what}: {int((over > 0).sum())} of {over.numel()} off, by {float(over.max()):.3g} at most, NaN {bool(torch.isnan(over).any())}"


SHAPES = [(1, 8, 16), (1, 4096, 1024), (3, 136, 144), (16, 128, 128), (17, 1000, 2048), (64, 1024, 4096), (65, 72, 272), (128, 256, 128), (200, 264, 400), (777, 1000, 1904),
          (2100, 1032, 1024), (300, 2304, 768), (4090, 4088, 400), (8190, 4088, 272)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K):
    print(f"gemm_q8 M={M} N={N} K={K}", flush=True)
    x, xs, w, ws = case(M, N, K, M + N + K, pad=16)
    xv, wv = values(M, N, K, x, xs, w, ws)
    want, terms = xv @ wv.t(), xv.abs() @ wv.abs().t()
    bound = ((K + 128) * 2.0 ** -23 + 2.0 ** -10) * terms
    near(run(M, N, K, x, xs, w, ws, ldy=N + 8), want, HALF * want.abs() + (1 + HALF) * bound, "Y")
    size = float(want.abs().mean())
    residual = (torch.randn(M, N + 8, generator=torch.Generator().manual_seed(M)) * size).to(BF16).cuda()
    total = want + residual[:, :N].double()
    added = run(M, N, K, x, xs, w, ws, residual=residual)
    near(added, total, HALF * total.abs() + (1 + HALF) * (bound + 2.0 ** -23 * total.abs()), "Y + residual")
    place = torch.empty(M, N, dtype=BF16, device="cuda").copy_(residual[:, :N])
    assert torch.equal(run(M, N, K, x, xs, w, ws, residual=place, out=place), added)


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_small_integers(M, N, K):
    """Integers up to 8 and scales that are powers of two: every sum is exact, and the result its one rounding."""
    g = torch.Generator().manual_seed(M * N + K)
    blocks = -(-K // 128)
    x = torch.randint(-8, 9, (M, K), generator=g).float().to(F8).view(torch.uint8).cuda()
    w = torch.randint(-8, 9, (N, K), generator=g).float().to(F8).view(torch.uint8).cuda()
    xs = torch.exp2(torch.randint(-2, 3, (blocks, M), generator=g).float()).cuda()
    ws = torch.exp2(torch.randint(-2, 3, (-(-N // 128), blocks), generator=g).float()).cuda()
    xv, wv = values(M, N, K, x, xs, w, ws)
    want = xv @ wv.t()
    assert float((xv.abs() @ wv.abs().t()).max()) < 2 ** 20  # of units of 2^-4: 24 bits
    assert torch.equal(run(M, N, K, x, xs, w, ws), want.to(BF16))


def test_every_code_stands_for_its_value():
    """x = one code in one place, w = one there: the outputs are the codes' values, NaN among them, in every place of a block."""
    for k in (0, 1, 31, 32, 63, 64, 100, 127, 128, 143):
        x = torch.zeros(256, 144, dtype=torch.uint8)
        x[:, k] = torch.arange(256)
        w = torch.zeros(8, 144, dtype=torch.uint8)
        w[:, k] = torch.tensor([1.0]).to(F8).view(torch.uint8)
        ones = torch.ones(2, 256, device="cuda")
        y = run(256, 8, 144, x.cuda(), ones, w.cuda(), torch.ones(1, 2, device="cuda"))
        want = x[:, k].view(F8).float()
        assert torch.equal(torch.nan_to_num(y.cpu().float(), nan=1e9), torch.nan_to_num(want, nan=1e9)[:, None].expand(256, 8))


def test_a_code_that_is_not_a_number_stays_in_its_row():
    x, xs, w, ws = case(300, 264, 400, 9)
    clean = run(300, 264, 400, x, xs, w, ws)
    x[33, 390] = 0x7f
    xs[1, 290] = float("inf")
    y = run(300, 264, 400, x, xs, w, ws)
    rest = torch.ones(300, dtype=torch.bool)
    rest[[33, 290]] = False
    assert bool(torch.isnan(y[33]).all()) and not bool(torch.isfinite(y[290]).any()) and torch.equal(y[rest], clean[rest])
