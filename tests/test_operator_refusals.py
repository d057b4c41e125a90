"""What the RMS norm, the quantisers, the 8-bit product and the gated block refuse: on the host, before anything is launched,
with the reason in tgk_error()."""
import pytest

from turbogpt_amd import bridge

A = 4096  # an aligned address that nothing reads: every call here is refused


def refused(call, needle):
    assert call == -1
    assert needle in bridge.library().tgk_error(), bridge.library().tgk_error()


def arguments(defaults, changes):
    return [changes.get(name, value) for name, value in defaults.items()]


NORM = dict(stream=None, rows=4, D=64, x=A, residual=A, hi=A, lo=A, sum=A, y=A, q=A, scales=A, ld_scales=4, eps=1e-6)
NORM_BACK = dict(stream=None, rows=4, D=64, x=A, dy=A, hi=A, lo=A, residual=A, dx=A, dgamma=A, eps=1e-6, accumulate=0, workspace=A, size=1 << 20)
ROWS = dict(stream=None, rows=4, columns=64, x=A, ldx=64, q=A, ldq=64, scales=A, ld_scales=4)
Q8 = dict(stream=None, M=4, N=64, K=256, X=A, ldx=256, xs=A, ldxs=4, W=A, ldw=256, ws=A, ldws=2, Y=A, ldy=64, residual=None, ldr=0)
GATED = dict(stream=None, M=4, F=64, D=32, X=A, ldx=32, W=A, ldw=32, H=A, ldh=64, GU=A, ldgu=128, act=0)
GATED_BACK = dict(stream=None, M=4, F=64, D=32, dY=A, lddy=32, Wdt=A, ldwdt=32, GU=A, ldgu=128, dGU=2 * A, lddgu=128, Wt=A, ldwt=128, dX=A, lddx=32, act=0)


HUGE = (1 << 30) + 1


@pytest.mark.parametrize("changes,needle", [
    (dict(rows=0), b"rows"), (dict(rows=HUGE, ld_scales=HUGE), b"rows"), (dict(D=0), b"multiple of 8"), (dict(D=12), b"multiple of 8"), (dict(D=8200), b"8192"), (dict(eps=-1.0), b"eps"),
    (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps"), (dict(x=None), b"x"), (dict(x=A + 2), b"aligned"), (dict(hi=None), b"gamma_hi"),
    (dict(lo=A + 8), b"gamma_lo"), (dict(residual=A + 2), b"residual"), (dict(sum=None), b"sum"), (dict(y=None, q=None), b"no output"),
    (dict(y=A + 8), b"y"), (dict(q=A + 4), b"q"), (dict(scales=None), b"scales"), (dict(ld_scales=3), b"ld_scales")])
def test_norm(changes, needle):
    refused(bridge.library().tgk_rmsnorm_fwd(*arguments(NORM, changes)), needle)


@pytest.mark.parametrize("changes,needle", [
    (dict(rows=-1), b"rows"), (dict(rows=HUGE), b"rows"), (dict(D=20), b"multiple of 8"), (dict(dy=None), b"dy"), (dict(dx=A + 2), b"dx"), (dict(dgamma=None), b"dgamma"),
    (dict(residual=A + 2), b"residual"), (dict(workspace=None), b"workspace"), (dict(workspace=A + 4), b"workspace"), (dict(size=64), b"workspace")])
def test_norm_backward(changes, needle):
    refused(bridge.library().tgk_rmsnorm_bwd(*arguments(NORM_BACK, changes)), needle)


def test_norm_workspace():
    lib = bridge.library()
    assert lib.tgk_rmsnorm_bwd_workspace(0, 64) == 0 and lib.tgk_rmsnorm_bwd_workspace(4, 0) == 0 and lib.tgk_rmsnorm_bwd_workspace(4, 8200) == 0
    assert lib.tgk_rmsnorm_bwd_workspace(1, 64) > 0


@pytest.mark.parametrize("changes,needle", [
    (dict(rows=0), b"row"), (dict(columns=12), b"columns"), (dict(x=None), b"x"), (dict(q=A + 4), b"q"), (dict(scales=None), b"scales"),
    (dict(ldx=56), b"leading"), (dict(ldx=68), b"leading"), (dict(ldq=56), b"leading"), (dict(ld_scales=3), b"ld_scales")])
def test_rows(changes, needle):
    refused(bridge.library().tgk_quantize_rows(*arguments(ROWS, changes)), needle)


@pytest.mark.parametrize("changes,needle", [
    (dict(rows=0), b"row"), (dict(columns=12), b"columns"), (dict(x=A + 2), b"w"), (dict(ldq=60), b"leading"), (dict(ld_scales=0), b"ld_scales")])
def test_weights(changes, needle):
    refused(bridge.library().tgk_quantize_tiles(*arguments(ROWS, changes)), needle)


@pytest.mark.parametrize("changes,needle", [
    (dict(M=0), b"M at least 1"), (dict(M=HUGE, ldxs=HUGE), b"at most"), (dict(N=1 << 30, ldy=1 << 30), b"Y"), (dict(N=60), b"multiple of 8"), (dict(K=264), b"multiple of 16"), (dict(K=0), b"K"), (dict(X=None), b"X"),
    (dict(X=A + 8), b"X"), (dict(ldx=264), b"X"), (dict(ldx=128), b"X"), (dict(W=A + 1), b"W"), (dict(ldw=1 << 23), b"W"), (dict(xs=None), b"x_scales"),
    (dict(ldxs=3), b"x_scales"), (dict(ws=A + 2), b"w_scales"), (dict(ldws=1), b"w_scales"), (dict(Y=None), b"Y"), (dict(ldy=60), b"Y"),
    (dict(residual=A + 2, ldr=64), b"residual"), (dict(residual=2 * A, ldr=32), b"residual"), (dict(residual=A, ldr=72), b"in place")])
def test_product(changes, needle):
    refused(bridge.library().tgk_gemm_q8(*arguments(Q8, changes)), needle)


@pytest.mark.parametrize("changes,needle", [
    (dict(M=0), b"M at least 1"), (dict(M=HUGE), b"at most"), (dict(F=60), b"multiples of 8"), (dict(D=4), b"multiples of 8"), (dict(act=2), b"activation"), (dict(act=-1), b"activation"),
    (dict(X=None), b"X"), (dict(ldx=24), b"X"), (dict(W=A + 2), b"W"), (dict(ldw=36), b"W"), (dict(H=None), b"H"), (dict(ldh=32), b"H"), (dict(ldgu=64), b"GU"),
    (dict(ldx=1 << 22), b"X")])
def test_gated(changes, needle):
    refused(bridge.library().tgk_gated_fwd(*arguments(GATED, changes)), needle)


@pytest.mark.parametrize("changes,needle", [
    (dict(M=0), b"M at least 1"), (dict(act=7), b"activation"), (dict(dY=None), b"dY"), (dict(Wdt=None), b"Wdt"), (dict(ldwdt=24), b"Wdt"), (dict(GU=None), b"GU"),
    (dict(ldgu=64), b"GU"), (dict(dGU=None), b"dGU"), (dict(dGU=A, lddgu=136), b"in place"), (dict(Wt=None), b"Wt"), (dict(ldwt=64), b"Wt"), (dict(dX=A + 2), b"dX"),
    (dict(lddx=24), b"dX")])
def test_gated_backward(changes, needle):
    refused(bridge.library().tgk_gated_bwd(*arguments(GATED_BACK, changes)), needle)
