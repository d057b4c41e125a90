"""The gated feed-forward block and its backward pass against the formulas in 64 bits.

Tolerances, element by element.  A product of K terms summed in 32 bits is off by at most K 2^-23 of the sum of the
terms' magnitudes (`slack`), a rounding to bfloat16 by 2^-8 of the value.  Activations and their slopes are evaluated to
2^-19 of 1 + |g| (an exponential and a reciprocal of 1 ulp each, the error function to 1.5e-7), and neither slope exceeds 1.13."""
import pytest
import torch

from gpu_util import check, library, stream, sync

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
SILU, GELU = 0, 1
HALF = 2.0 ** -8
ACT = 2.0 ** -19
SHAPES = [(1, 8, 8), (1, 256, 128), (2, 1720, 640), (17, 72, 200), (64, 64, 64), (65, 136, 72), (128, 256, 128), (129, 264, 192), (333, 1720, 640), (700, 520, 1000),
          (2048, 1024, 256), (12400, 1024, 136), (6272, 2048, 384)]


def slack(a, b):
    """K 2^-23 of the sum of magnitudes of a b^T."""
    return (a.double().abs() @ b.double().abs().t()) * (a.shape[1] * 2.0 ** -23)


def product(a, b):
    return a.double() @ b.double().t()


def act_and_slope(g, which):
    if which == SILU:
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g)
    phi = torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    cdf = 0.5 * torch.erfc(-g / 2 ** 0.5)
    return g * cdf, cdf + g * phi


def near(got, want, bound, what):
    over = (got.double() - want).abs() - bound
    assert bool((over <= 0).all()), f"{what}: {int((over > 0).sum())} of {over.numel()} off, by {float(over.max()):.3g} at most, NaN {bool(torch.isnan(over).any())}"


def padded(rows, columns, ld, generator, scale=1.0):
    """A view [rows][columns] of a matrix with wider rows, NaN behind them."""
    whole = torch.full((rows, ld), float("nan"))
    whole[:, :columns] = torch.randn(rows, columns, generator=generator) * scale
    return whole.to(BF16).cuda()[:, :columns]


def blank(rows, columns, ld):
    return torch.full((rows + 2, ld), 7.0, dtype=BF16, device="cuda")


def untouched(whole, rows, columns):
    return bool((whole[rows:] == 7.0).all()) and bool((whole[:, columns:] == 7.0).all())


def forward(x, w, act, keep, ldh=None, ldgu=None):
    (M, D), F = x.shape, w.shape[0] // 2
    ldh, ldgu = ldh or F, ldgu or 2 * F
    h, gu = blank(M, F, ldh), blank(M, 2 * F, ldgu)
    check(library().tgk_gated_fwd(stream(), M, F, D, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), h.data_ptr(), ldh,
                                  gu.data_ptr() if keep else None, ldgu, act))
    sync()
    assert untouched(h, M, F) and untouched(gu, M if keep else 0, 2 * F)
    return h[:M, :F], gu[:M, :2 * F]


def check_forward(x, w, h, gu, act):
    F = w.shape[0] // 2
    both, off = product(x, w), slack(x, w)
    g, u = both[:, :F], both[:, F:]
    a, _ = act_and_slope(g, act)
    first = 1.13 * off[:, :F] + ACT * (1 + g.abs())
    near(h, a * u, HALF * (a * u).abs() + (1 + HALF) * (first * (u.abs() + off[:, F:]) + a.abs() * off[:, F:]) + 1e-38, "H")
    if gu is not None:
        near(gu, both, HALF * both.abs() + (1 + HALF) * off + 1e-38, "GU")


@pytest.mark.parametrize("act", [SILU, GELU])
@pytest.mark.parametrize("M,F,D", SHAPES)
def test_forward(M, F, D, act):
    print(f"gated_fwd M={M} F={F} D={D} act={act}", flush=True)
    g = torch.Generator().manual_seed(M + F + D)
    x, w = padded(M, D, D + 8, g), padded(2 * F, D, D + 16, g, D ** -0.5)
    h, gu = forward(x, w, act, True, F + 8, 2 * F + 24)
    check_forward(x, w, h, gu, act)
    alone, _ = forward(x, w, act, False)
    assert torch.equal(alone, h)


def backward(dy, wdt, gu, wt, act, want_dx=True, in_place=False):
    M, D = dy.shape
    F = wdt.shape[0]
    if in_place:
        dgu = gu
        ld = gu.stride(0)
    else:
        ld = 2 * F + 8
        dgu = blank(M, 2 * F, ld)
    dx = blank(M, D, D + 8)
    check(library().tgk_gated_bwd(stream(), M, F, D, dy.data_ptr(), dy.stride(0), wdt.data_ptr(), wdt.stride(0), gu.data_ptr(), gu.stride(0),
                                  dgu.data_ptr(), ld, wt.data_ptr() if want_dx else None, wt.stride(0), dx.data_ptr() if want_dx else None, D + 8, act))
    sync()
    assert in_place or untouched(dgu, M, 2 * F)
    assert untouched(dx, M if want_dx else 0, D)
    return dgu[:M, :2 * F], dx[:M, :D]


@pytest.mark.parametrize("act", [SILU, GELU])
@pytest.mark.parametrize("M,F,D", SHAPES)
def test_backward(M, F, D, act):
    print(f"gated_bwd M={M} F={F} D={D} act={act}", flush=True)
    g = torch.Generator().manual_seed(M + F + D + 1)
    dy, wdt = padded(M, D, D + 8, g), padded(F, D, D + 8, g, F ** -0.5)
    gu, wt = padded(M, 2 * F, 2 * F + 8, g, 1.5), padded(D, 2 * F, 2 * F + 16, g, D ** -0.5)
    dgu, dx = backward(dy, wdt, gu, wt, act)
    dh, off = product(dy, wdt), slack(dy, wdt)
    gate, up = gu.double()[:, :F], gu.double()[:, F:]
    a, slope = act_and_slope(gate, act)
    loose = ACT * (1 + gate.abs())
    want = torch.cat([dh * up * slope, dh * a], 1)
    bound = torch.cat([up.abs() * (1.13 * off + (dh.abs() + off) * loose), a.abs() * off + (dh.abs() + off) * loose], 1)
    near(dgu, want, HALF * want.abs() + (1 + HALF) * bound + 1e-38, "dGU")
    want = product(dgu, wt)
    near(dx, want, HALF * want.abs() + (1 + HALF) * slack(dgu, wt) + 1e-38, "dX")
    alone, _ = backward(dy, wdt, gu, wt, act, want_dx=False)
    assert torch.equal(alone, dgu)
    placed, again = backward(dy, wdt, gu.clone(), wt, act, in_place=True)
    assert torch.equal(placed, dgu) and torch.equal(again, dx)


def test_what_is_not_finite_stays_in_its_row():
    g = torch.Generator().manual_seed(3)
    x, w = padded(200, 136, 136, g), padded(2 * 96, 136, 136, g, 0.1)
    clean, _ = forward(x, w, SILU, False)
    x[7, 20], x[150, 135] = float("nan"), float("inf")
    h, gu = forward(x, w, SILU, True)
    rest = torch.ones(200, dtype=torch.bool)
    rest[[7, 150]] = False
    assert bool(torch.isnan(h[7]).all()) and not bool(torch.isfinite(gu[150]).any()) and torch.equal(h[rest], clean[rest])


@pytest.mark.parametrize("act", [SILU, GELU])
def test_far_gates(act):
    """Gates of hundreds either way: the activation is the gate or nothing, its slope one or nothing."""
    x = torch.tensor([[300.0], [-300.0], [80.0], [-80.0]], dtype=BF16).expand(4, 8).contiguous().cuda()
    x[:, 1:] = 0
    w = torch.zeros(16, 8, dtype=BF16, device="cuda")
    w[:8, 0], w[8:, 0] = 1.0, 1.0
    h, gu = forward(x, w, act, True)
    want = torch.tensor([90112.0, 0.0, 6400.0, 0.0]).to(BF16).double()  # 300^2 rounds to 90112
    assert float((h.cpu().double().abs() - want[:, None]).abs().max()) < 1e-30
    dy = torch.ones(4, 8, dtype=BF16, device="cuda")
    wdt = torch.zeros(8, 8, dtype=BF16, device="cuda")
    wdt[:, 0] = 1
    dgu, _ = backward(dy, wdt, gu, w.t().contiguous(), act)
    gate = torch.tensor([300.0, -300.0, 80.0, -80.0])
    on = (gate > 0).double()
    for column in (0, 8):
        assert float((dgu[:, column].cpu().double().abs() - gate.abs() * on).abs().max()) < 1e-30


def test_gradients_of_the_block_against_differences():
    """The block's own gradients, weights included, against central differences of its formula in 64 bits.  The backward pass
    rounds G, U, dG and dU to bfloat16: sums over them are off by 3 x 2^-8 of their terms' magnitudes at most."""
    g = torch.Generator().manual_seed(4)
    M, F, D = 32, 128, 128
    x, w, wd = padded(M, D, D, g), padded(2 * F, D, D, g, D ** -0.5), padded(D, F, F, g, F ** -0.5)
    dy = padded(M, D, D, g)
    _, gu = forward(x, w, SILU, True)
    gu = gu.contiguous()
    dgu, dx = backward(dy, wd.t().contiguous(), gu, w.t().contiguous(), SILU)
    dgu = dgu.contiguous()
    dw = torch.empty(2 * F, D, device="cuda")
    need = library().tgk_gemm_wgrad_workspace(M, 2 * F, D)
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    check(library().tgk_gemm_wgrad(stream(), M, 2 * F, D, dgu.data_ptr(), 2 * F, x.data_ptr(), D, dw.data_ptr(), D, 0, workspace.data_ptr(), need))
    sync()

    def loss(x, w):
        both = x @ w.t()
        return ((act_and_slope(both[:, :F], SILU)[0] * both[:, F:]) @ wd.double().t() * dy.double()).sum()

    step, x64, w64 = 1e-4, x.double(), w.double()
    terms_x, terms_w = dgu.double().abs() @ w64.abs(), dgu.double().abs().t() @ x64.abs()
    for r, c in [(0, 0), (5, 77), (31, 127)]:
        e = torch.zeros_like(x64)
        e[r, c] = step
        slope = float(loss(x64 + e, w64) - loss(x64 - e, w64)) / (2 * step)
        assert abs(float(dx[r, c]) - slope) <= 3 * HALF * float(terms_x[r, c]) + 1e-5
    for r, c in [(3, 9), (127, 0), (128, 5), (255, 127)]:
        e = torch.zeros_like(w64)
        e[r, c] = step
        slope = float(loss(x64, w64 + e) - loss(x64, w64 - e)) / (2 * step)
        assert abs(float(dw[r, c]) - slope) <= 3 * HALF * float(terms_w[r, c]) + 1e-5
