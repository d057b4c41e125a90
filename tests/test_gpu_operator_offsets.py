"""Operands of more than 2^32 bytes: what rows far apart, or many rows, give is, bit for bit, what the same rows give side by side."""
import pytest
import torch

from gpu_util import check, library, stream, sync

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
FAR = 1 << 21  # the largest leading dimension in elements of 16 bits; twice that in codes
FAR_BYTES = 1 << 32


def apart(values, ld):
    """The same rows, `ld` elements apart; nothing is written between them."""
    far = torch.empty(values.shape[0] * ld, dtype=values.dtype, device="cuda").view(values.shape[0], ld)[:, :values.shape[1]]
    far.copy_(values)
    assert (values.shape[0] - 1) * ld * values.element_size() > FAR_BYTES
    return far


def room(rows, columns, ld, dtype=BF16):
    return torch.empty(rows * ld, dtype=dtype, device="cuda").view(rows, ld)[:, :columns]


def normal(rows, columns, seed, scale=1.0):
    return (torch.randn(rows, columns, generator=torch.Generator().manual_seed(seed)) * scale).to(BF16).cuda()


@pytest.mark.parametrize("M,N,K", [(1100, 64, 272), (1100, 1096, 272), (2100, 4088, 2048)])  # blocks that share out k, small tiles, large ones
def test_product_of_codes(M, N, K):
    blocks = -(-K // 128)
    g = torch.Generator().manual_seed(N)
    x, w = (torch.randint(0, 0x7f, (rows, K), generator=g, dtype=torch.uint8).cuda() for rows in (M, N))
    xs, ws = torch.rand(blocks, M, generator=g).cuda(), torch.rand(-(-N // 128), blocks, generator=g).cuda()
    residual = normal(M, N, N + 1)

    def run(x, w, residual, y):
        check(library().tgk_gemm_q8(stream(), M, N, K, x.data_ptr(), x.stride(0), xs.data_ptr(), M, w.data_ptr(), w.stride(0), ws.data_ptr(), blocks,
                                    y.data_ptr(), y.stride(0), residual.data_ptr(), residual.stride(0)))
        sync()
        return y

    want = run(x, w, residual, torch.empty(M, N, dtype=BF16, device="cuda"))
    got = run(apart(x, 2 * FAR), apart(w, 2 * FAR) if N > 1024 else w, apart(residual, FAR), room(M, N, FAR))
    assert bool(torch.isfinite(want).all()) and torch.equal(got, want)


@pytest.mark.parametrize("M,D,F", [(1100, 72, 528), (1152, 128, 528), (1100, 16, 16), (2100, 1024, 1416)])  # dX by either product; blocks that share out k; large tiles
def test_gated_block(M, D, F):
    x, w, dy = normal(M, D, 1), normal(2 * F, D, 2, D ** -0.5), normal(M, D, 3)
    wdt, wt = normal(F, D, 4, F ** -0.5), normal(D, 2 * F, 5, D ** -0.5)

    def run(x, w, dy, h, gu, dgu, dx):
        check(library().tgk_gated_fwd(stream(), M, F, D, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), h.data_ptr(), h.stride(0), gu.data_ptr(),
                                      gu.stride(0), 0))
        check(library().tgk_gated_bwd(stream(), M, F, D, dy.data_ptr(), dy.stride(0), wdt.data_ptr(), D, gu.data_ptr(), gu.stride(0), dgu.data_ptr(),
                                      dgu.stride(0), wt.data_ptr(), 2 * F, dx.data_ptr(), dx.stride(0), 0))
        sync()
        return h, gu, dgu, dx

    widths = (F, 2 * F, 2 * F, D)
    want = run(x, w, dy, *(room(M, columns, columns) for columns in widths))
    got = run(apart(x, FAR), apart(w, FAR) if 2 * F > 1024 else w, apart(dy, FAR), *(room(M, columns, FAR) for columns in widths))
    for name, a, b in zip(("H", "GU", "dGU", "dX"), got, want):
        assert bool(torch.isfinite(b).all()) and torch.equal(a, b), name


def test_rows_to_codes():
    rows, columns = 1100, 264
    x = normal(rows, columns, 7)

    def run(x, q):
        scales = torch.empty(3, rows, device="cuda")
        check(library().tgk_quantize_rows(stream(), rows, columns, x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), scales.data_ptr(), rows))
        tiles = torch.empty(-(-rows // 128), 3, device="cuda")
        sync()
        by_row = q.clone()
        check(library().tgk_quantize_tiles(stream(), rows, columns, x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), tiles.data_ptr(), 3))
        sync()
        return by_row, scales, q, tiles

    want = run(x, room(rows, columns, columns, torch.uint8))
    got = run(apart(x, FAR), room(rows, columns, 2 * FAR, torch.uint8))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_norm_of_many_rows():
    """The last rows of 2^31 + 2^15 values by themselves: each row's results are its own.  Only these rows have a gradient, so that dgamma is theirs too, but
    added in another order: off by the last bits of terms that are summed in 32 bits."""
    D, last = 8192, 8
    rows = (1 << 18) + 4
    x, residual = torch.ones(rows, D, dtype=BF16, device="cuda"), torch.ones(rows, D, dtype=BF16, device="cuda")
    dy = torch.zeros(rows, D, dtype=BF16, device="cuda")
    x[-last:], residual[-last:], dy[-last:] = normal(last, D, 1), normal(last, D, 2), normal(last, D, 3)
    bits = (1 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(4))).cuda().view(torch.int32)
    hi, lo = (bits >> 16).to(torch.int16), (bits & 0xffff).to(torch.int16)

    def run(x, residual, dy):
        n = x.shape[0]
        total, y, dx = (torch.empty(n, D, dtype=BF16, device="cuda") for _ in range(3))
        q, scales = torch.empty(n, D, dtype=torch.uint8, device="cuda"), torch.empty(D // 128, n, device="cuda")
        check(library().tgk_rmsnorm_fwd(stream(), n, D, x.data_ptr(), residual.data_ptr(), hi.data_ptr(), lo.data_ptr(), total.data_ptr(), y.data_ptr(),
                                        q.data_ptr(), scales.data_ptr(), n, 1e-6))
        need = library().tgk_rmsnorm_bwd_workspace(n, D)
        workspace, dgamma = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty(D, device="cuda")
        check(library().tgk_rmsnorm_bwd(stream(), n, D, total.data_ptr(), dy.data_ptr(), hi.data_ptr(), lo.data_ptr(), residual.data_ptr(), dx.data_ptr(),
                                        dgamma.data_ptr(), 1e-6, 0, workspace.data_ptr(), need))
        sync()
        return [t[-last:] for t in (total, y, q, dx)] + [scales[:, -last:]], dgamma

    got, got_gamma = run(x, residual, dy)
    want, want_gamma = run(x[-last:].contiguous(), residual[-last:].contiguous(), dy[-last:].contiguous())
    for name, a, b in zip(("sum", "y", "codes", "dx", "scales"), got, want):
        assert torch.equal(a, b), name
    # eight terms, seven additions on either side, each off by 2^-24 of what it adds up: 14 x 2^-24 of the magnitudes, under 2^-20; the terms
    # themselves are the same on both sides
    h = want[0].double()
    terms = (dy[-last:].double() * h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6)).abs().sum(0)
    assert bool(torch.isfinite(want_gamma).all())
    assert bool(((got_gamma - want_gamma).double().abs() <= terms * 2.0 ** -20).all())
