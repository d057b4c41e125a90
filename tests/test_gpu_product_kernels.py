"""Every kernel of the products of any shape, with every epilogue, with one tile a block and with several, and with a single stage of k, against
the definitions in 64 bits: the checks of test_gpu_gated.py and test_gpu_gemm_q8.py, whose tolerances hold at any size, on shapes that the rule sends
to each.  test_product_rules.py asks the rule whether they still do."""
import pytest
import torch

import test_gpu_gated as gated
import test_gpu_gemm_q8 as q8

pytestmark = pytest.mark.gpu

# M, F, D
GATED = [(3001, 40, 136), (49, 1040, 144), (8428, 72, 64), (7219, 1704, 24), (5063, 528, 304), (10954, 656, 40), (10968, 272, 56), (7314, 1352, 720),
         (3578, 3272, 136), (13161, 264, 584), (11019, 3744, 720), (13384, 32, 528), (12701, 16, 936), (15001, 264, 2040)]
# M, N, K
Q8 = [(49, 1040, 144), (2048, 256, 1024), (512, 1024, 1024), (8530, 72, 112), (5726, 208, 272), (11006, 648, 128), (7000, 1000, 208), (11674, 800, 16),
      (6752, 2360, 656)]


@pytest.mark.parametrize("act", [gated.SILU, gated.GELU])
@pytest.mark.parametrize("M,F,D", GATED)
def test_gated_forward(M, F, D, act):
    gated.test_forward(M, F, D, act)


@pytest.mark.parametrize("act", [gated.SILU, gated.GELU])
@pytest.mark.parametrize("M,F,D", GATED)
def test_gated_backward(M, F, D, act):
    gated.test_backward(M, F, D, act)


@pytest.mark.parametrize("M,N,K", Q8)
def test_product_of_codes(M, N, K):
    q8.test_product(M, N, K)


@pytest.mark.parametrize("M,N,K", Q8)
def test_small_integers(M, N, K):
    q8.test_small_integers(M, N, K)


# Powers of two of a row's and a tile's scale, which are up to twice that: their product is a normal number.
@pytest.mark.parametrize("rows,tiles", [(-100, -26), (-26, -100), (-63, -63), (-100, 100), (110, -100), (-1, -100)])
@pytest.mark.parametrize("M,N,K", [(1, 8, 16), (49, 1040, 144), (2048, 256, 272), (777, 1000, 400), (5726, 208, 272), (7000, 1000, 208), (4090, 4088, 272)])
def test_scales_far_from_one(M, N, K, rows, tiles):
    """As test_product; the block's sums times a product of scales of 2^-126 or more are added in 32 bits, off by half a subnormal step, 2^-150, each; the
    result's rounding is off by half of bfloat16's step, 2^-134, among its subnormal values."""
    g = torch.Generator().manual_seed(M + N + K)
    x, _, w, _ = q8.case(M, N, K, M + N + K)
    blocks = -(-K // 128)
    xs = (2.0 ** rows * (1 + torch.rand(blocks, M, generator=g))).cuda()
    ws = (2.0 ** tiles * (1 + torch.rand(-(-N // 128), blocks, generator=g))).cuda()
    xv, wv = q8.values(M, N, K, x, xs, w, ws)
    want, terms = xv @ wv.t(), xv.abs() @ wv.abs().t()
    bound = ((K + 128) * 2.0 ** -23 + 2.0 ** -10) * terms + blocks * 2.0 ** -150
    q8.near(q8.run(M, N, K, x, xs, w, ws), want, q8.HALF * want.abs() + (1 + q8.HALF) * bound + 2.0 ** -134, "Y")
