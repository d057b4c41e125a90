"""RMS norm with the residual's addition, its 8-bit output and its backward pass, and the quantisers, against the
definitions in 64 bits.

Tolerances.  A rounding to bfloat16 is off by at most 2^-8 of the value, to e4m3 by 2^-4 of it or half of the step 2^-9
among the subnormal codes.  What is computed in 32 bits first (a sum of squares of at most 8192 terms over 64 lanes or
more, a root, a quotient, three products) is off by less than (8192 / 64 + 32) 2^-24 < 2^-16 of its terms."""
import numpy as np
import pytest
import torch

from gpu_util import check, library, stream, sync

pytestmark = pytest.mark.gpu

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
FP32 = 2.0 ** -16
LEAST = 2.0 ** -100
EPS = 1e-6


def halves(gamma):
    bits = gamma.view(torch.int32)
    return (bits >> 16).to(torch.int16), (bits & 0xffff).to(torch.int16)


def groups(v):
    """Largest magnitudes [rows][ceil(columns / 128)] of rows, in the rows' type."""
    wide = torch.nn.functional.pad(v, (0, -v.shape[1] % 128))
    return wide.view(v.shape[0], -1, 128).abs().amax(2)


def per_column(scales, columns):
    return scales.repeat_interleave(128, 1)[:, :columns]


def near(got, want, bound, what):
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), f"{what}: {int((over > 0).sum())} of {over.numel()} off, by {float(over.max()):.3g} at most"


def inputs(rows, D, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, D, generator=g) * 2).to(BF16).cuda()
    residual = torch.randn(rows, D, generator=g).to(BF16).cuda()
    gamma = (1 + 0.2 * torch.randn(D, generator=g)).cuda()
    return x, residual, gamma


def forward(x, residual, gamma, want_y=True, want_q=True, into=None, guard=5):
    """Outputs with `guard` rows behind the last, which have to stay as they were."""
    rows, D = x.shape
    hi, lo = halves(gamma)
    total = torch.full((rows + guard, D), 7.0, dtype=BF16, device="cuda") if into is None else into
    y = torch.full((rows + guard, D), 7.0, dtype=BF16, device="cuda")
    q = torch.full((rows + guard, D), 0x55, dtype=torch.uint8, device="cuda")
    ld = rows + 3
    scales = torch.full((-(-D // 128), ld), 7.0, device="cuda")
    check(library().tgk_rmsnorm_fwd(stream(), rows, D, x.data_ptr(), residual.data_ptr() if residual is not None else None, hi.data_ptr(),
                                    lo.data_ptr(), total.data_ptr() if residual is not None else None, y.data_ptr() if want_y else None,
                                    q.data_ptr() if want_q else None, scales.data_ptr() if want_q else None, ld, EPS))
    sync()
    if into is None and residual is not None:
        assert bool((total[rows:] == 7.0).all())
    assert bool((y[rows if want_y else 0:] == 7.0).all()) and bool((q[rows if want_q else 0:] == 0x55).all())
    assert bool((scales[:, rows if want_q else 0:] == 7.0).all())
    return total[:rows], y[:rows], q[:rows].view(F8), scales[:, :rows]


def normalised(h, gamma):
    h = h.double()
    return h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * gamma.double()


def check_codes(q, scales, v):
    want = (groups(v) / 448).clamp(min=LEAST)
    near(scales.t(), want, want * FP32, "scales")
    scale = per_column(scales.t().double(), v.shape[1])
    near(q.double() * scale, v, v.abs() * (2.0 ** -4 + FP32) + scale * 2.0 ** -10, "codes")


@pytest.mark.parametrize("rows,D", [(1, 8), (3, 1024), (5, 120), (33, 136), (64, 512), (17, 520), (130, 1000), (6, 2048), (5, 2056), (9, 8192), (4100, 768), (8500, 2048)])
def test_forward(rows, D):
    x, residual, gamma = inputs(rows, D, rows * 8192 + D)
    total, y, q, scales = forward(x, residual, gamma)
    h = (x.float() + residual.float()).to(BF16)
    assert torch.equal(total, h)
    v = normalised(h, gamma)
    near(y, v, v.abs() * (2.0 ** -8 + FP32), "y")
    check_codes(q, scales, v)


def test_outputs_one_by_one_and_without_a_residual():
    x, residual, gamma = inputs(19, 264, 1)
    _, y, q, scales = forward(x, residual, gamma)
    _, only_y, _, _ = forward(x, residual, gamma, want_q=False)
    _, _, only_q, only_scales = forward(x, residual, gamma, want_y=False)
    assert torch.equal(y, only_y) and torch.equal(q.view(torch.uint8), only_q.view(torch.uint8)) and torch.equal(scales, only_scales)
    _, y, _, _ = forward(x, None, gamma)
    v = normalised(x, gamma)
    near(y, v, v.abs() * (2.0 ** -8 + FP32), "y")


@pytest.mark.parametrize("which", ["x", "residual"])
def test_the_sum_in_place(which):
    x, residual, gamma = inputs(40, 768, 2)
    total, y, _, _ = forward(x, residual, gamma)
    a, b = x.clone(), residual.clone()
    place = a if which == "x" else b
    _, again, _, _ = forward(a, b, gamma, into=place)
    assert torch.equal(place, total) and torch.equal(again, y)


def test_rows_of_zeros_small_values_and_what_is_not_finite():
    x, _, gamma = inputs(6, 384, 3)
    x[0] = 0
    x[1] = x[1] * 1e-30
    x[2, 200] = float("nan")
    x[3, 5] = float("inf")
    _, y, q, scales = forward(x, None, gamma)
    assert bool((y[0] == 0).all()) and bool((q[0].float() == 0).all()) and bool((scales[:, 0] == np.float32(LEAST)).all())
    assert bool((y[1].float().abs() < 1e-20).all()) and bool(torch.isfinite(scales[:, 1]).all())
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(q[2].float()).all())
    assert bool(torch.isnan(y[3, 5])) and bool((y[3, 6:] == 0).all())
    v = normalised(x[4:], gamma)
    near(y[4:], v, v.abs() * (2.0 ** -8 + FP32), "y")
    check_codes(q[4:], scales[:, 4:], v)


def backward(h, dy, gamma, residual, dgamma=None, in_place=False):
    rows, D = h.shape
    hi, lo = halves(gamma)
    dx = residual.clone() if in_place else torch.full((rows + 2, D), 7.0, dtype=BF16, device="cuda")
    out = torch.full((D,), 9.0, device="cuda") if dgamma is None else dgamma.clone()
    need = library().tgk_rmsnorm_bwd_workspace(rows, D)
    workspace = torch.full((need + 16,), 0x7f, dtype=torch.uint8, device="cuda")
    check(library().tgk_rmsnorm_bwd(stream(), rows, D, h.data_ptr(), dy.data_ptr(), hi.data_ptr(), lo.data_ptr(),
                                    dx.data_ptr() if in_place else residual.data_ptr() if residual is not None else None, dx.data_ptr(),
                                    out.data_ptr(), EPS, 0 if dgamma is None else 1, workspace.data_ptr(), need))
    sync()
    assert bool((workspace[need:] == 0x7f).all())
    if not in_place:
        assert bool((dx[rows:] == 7.0).all())
    return dx[:rows], out


def exact_backward(h, dy, gamma):
    h, dy, gamma = h.double(), dy.double(), gamma.double()
    D = h.shape[1]
    s = 1 / torch.sqrt(h.square().mean(1, keepdim=True) + EPS)
    t = dy * gamma
    pull = (h * t).sum(1, keepdim=True) * s ** 2 / D
    terms = s * (t.abs() + h.abs() * (h * t).abs().sum(1, keepdim=True) * s ** 2 / D)
    return s * (t - h * pull), terms, (dy * h * s).sum(0), (dy * h * s).abs().sum(0)


@pytest.mark.parametrize("rows,D", [(1, 8), (2, 1024), (7, 136), (65, 512), (130, 1000), (12, 2048), (11, 2056), (5, 8192), (6500, 768), (8500, 2048)])
def test_backward(rows, D):
    h, residual, gamma = inputs(rows, D, rows * 8192 + D + 1)
    dy = torch.randn(rows, D, generator=torch.Generator().manual_seed(rows)).to(BF16).cuda()
    dv, terms, dgamma, sums = exact_backward(h, dy, gamma)
    dx, got = backward(h, dy, gamma, residual)
    want = residual.double() + dv
    near(dx, want, (2.0 ** -8 + FP32) * want.abs() + terms * FP32, "dx")
    near(got, dgamma, sums * FP32, "dgamma")
    plain, _ = backward(h, dy, gamma, None)
    near(plain, dv, (2.0 ** -8 + FP32) * dv.abs() + terms * FP32, "dx without a residual")
    placed, again = backward(h, dy, gamma, residual, in_place=True)
    assert torch.equal(placed, dx) and torch.equal(again, got)
    start = torch.randn(D, generator=torch.Generator().manual_seed(D)).cuda()
    _, added = backward(h, dy, gamma, residual, dgamma=start)
    assert torch.equal(added, start + got)


def test_gradient_against_differences():
    """Central differences of the formula in 64 bits, weighted by dy: off by step^2 times a third derivative of order 1."""
    h, _, gamma = inputs(2, 24, 5)
    dy = torch.randn(2, 24, generator=torch.Generator().manual_seed(6)).to(BF16).cuda()
    dx, dgamma = backward(h, dy, gamma, None)
    step, h64, g64 = 1e-4, h.double(), gamma.double()
    at = lambda a, b: (a / torch.sqrt(a.square().mean(1, keepdim=True) + EPS) * b * dy.double()).sum()  # noqa: E731
    for r, c in [(0, 0), (0, 13), (1, 7), (1, 23)]:
        e = torch.zeros_like(h64)
        e[r, c] = step
        slope = float(at(h64 + e, g64) - at(h64 - e, g64)) / (2 * step)
        assert abs(float(dx[r, c]) - slope) <= 2.0 ** -8 * abs(slope) + 1e-5
    e = torch.zeros_like(g64)
    e[11] = step
    assert abs(float(dgamma[11]) - float(at(h64, g64 + e) - at(h64, g64 - e)) / (2 * step)) <= 1e-4


@pytest.mark.parametrize("rows,columns,ldx,ldq", [(1, 8, 8, 8), (5, 128, 136, 144), (33, 1000, 1000, 1008), (70, 512, 520, 512), (3, 4104, 4104, 4112), (9000, 136, 136, 136)])
def test_rows_to_codes(rows, columns, ldx, ldq):
    """Codes and scales are those of the definition in 32 bits, bit for bit: one quotient each, rounded once."""
    g = torch.Generator().manual_seed(rows + columns)
    x = (torch.randn(rows, ldx, generator=g) * torch.exp(4 * torch.randn(rows, 1, generator=g))).to(BF16).cuda()
    if rows > 2:
        x[1, :columns] = 0
        x[2, :columns] = 1e-38
    q = torch.full((rows + 1, ldq), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((-(-columns // 128), rows + 2), 7.0, device="cuda")
    check(library().tgk_quantize_rows(stream(), rows, columns, x.data_ptr(), ldx, q.data_ptr(), ldq, scales.data_ptr(), rows + 2))
    sync()
    v = x[:, :columns].float().cpu()
    want = (groups(v) / 448).clamp(min=LEAST)
    assert torch.equal(scales[:, :rows].t().cpu(), want) and bool((scales[:, rows:] == 7.0).all())
    assert torch.equal(q[:rows, :columns].cpu(), (v / per_column(want, columns)).to(F8).view(torch.uint8))
    assert bool((q[rows:] == 0x55).all()) and bool((q[:, columns:] == 0x55).all())


@pytest.mark.parametrize("rows,columns", [(1, 8), (128, 128), (130, 136), (1000, 264), (300, 1920)])
def test_weights_to_codes(rows, columns):
    g = torch.Generator().manual_seed(rows * columns)
    ld = columns + 16
    w = (torch.randn(rows, ld, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(BF16).cuda()
    tiles_m, tiles_n = -(-rows // 128), -(-columns // 128)
    q = torch.full((rows + 1, ld), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((tiles_m, tiles_n + 1), 7.0, device="cuda")
    check(library().tgk_quantize_tiles(stream(), rows, columns, w.data_ptr(), ld, q.data_ptr(), ld, scales.data_ptr(), tiles_n + 1))
    sync()
    v = w[:, :columns].float().cpu()
    padded = torch.nn.functional.pad(v, (0, -columns % 128, 0, -rows % 128)).view(tiles_m, 128, tiles_n, 128)
    want = (padded.abs().amax((1, 3)) / 448).clamp(min=LEAST)
    assert torch.equal(scales[:, :tiles_n].cpu(), want) and bool((scales[:, tiles_n:] == 7.0).all())
    full = want.repeat_interleave(128, 0).repeat_interleave(128, 1)[:rows, :columns]
    assert torch.equal(q[:rows, :columns].cpu(), (v / full).to(F8).view(torch.uint8))
    assert bool((q[rows:] == 0x55).all()) and bool((q[:, columns:] == 0x55).all())


def test_what_is_not_finite_in_rows_to_codes():
    x = torch.randn(3, 256, generator=torch.Generator().manual_seed(8)).to(BF16).cuda()
    x[0, 3], x[1, 130] = float("nan"), float("-inf")
    q = torch.empty(3, 256, dtype=F8, device="cuda")
    scales = torch.empty(2, 3, device="cuda")
    check(library().tgk_quantize_rows(stream(), 3, 256, x.data_ptr(), 256, q.data_ptr(), 256, scales.data_ptr(), 3))
    sync()
    stands_for = (q.float() * per_column(scales.t(), 256)).cpu()
    nan = torch.isnan(stands_for)
    assert bool(nan[0, 3]) and int(nan[0].sum()) == 1 and bool(nan[1, 128:].all()) and not bool(nan[1, :128].any()) and not bool(nan[2].any())
