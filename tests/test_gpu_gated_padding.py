"""A batch padded with rows of zeros, as the products around the gated block want it: the padding's results and gradients are zeros, and the
weights' gradients are those of the batch alone."""
import pytest
import torch

import test_gpu_gated as gated
from gpu_util import check, library, stream, sync

pytestmark = pytest.mark.gpu


def weight_gradient(dgu, x):
    (M, N), K = dgu.shape, x.shape[1]
    dw = torch.empty(N, K, device="cuda")
    need = library().tgk_gemm_wgrad_workspace(M, N, K)
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    check(library().tgk_gemm_wgrad(stream(), M, N, K, dgu.data_ptr(), N, x.data_ptr(), K, dw.data_ptr(), K, 0, workspace.data_ptr(), need))
    sync()
    return dw


@pytest.mark.parametrize("act", [gated.SILU, gated.GELU])
@pytest.mark.parametrize("M,padded,F,D", [(1, 128, 192, 128), (333, 384, 256, 384), (1100, 1152, 320, 128)])
def test_rows_of_zeros_add_nothing(M, padded, F, D, act):
    g = torch.Generator().manual_seed(M)
    x, dy = gated.padded(padded, D, D, g), gated.padded(padded, D, D, g)
    x[M:], dy[M:] = 0, 0
    w, wdt = gated.padded(2 * F, D, D, g, D ** -0.5), gated.padded(F, D, D, g, F ** -0.5)
    wt = w.t().contiguous()
    h, gu = gated.forward(x, w, act, True)
    gu = gu.contiguous()
    dgu, dx = (t.contiguous() for t in gated.backward(dy, wdt, gu, wt, act))
    for name, t in (("H", h), ("GU", gu), ("dGU", dgu), ("dX", dx)):
        assert bool((t[M:] == 0).all()), name
    dw = weight_gradient(dgu, x)
    want, terms = dgu[:M].double().t() @ x[:M].double(), dgu[:M].double().abs().t() @ x[:M].double().abs()
    gated.near(dw, want, terms * padded * 2.0 ** -23 + 1e-38, "dW")
