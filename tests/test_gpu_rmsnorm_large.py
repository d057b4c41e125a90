"""RMS norms whose results are larger than 32 MiB, which go past the L2s by kernels of their own, at every width's kernel, with and without a residual;
rows of more than 2048 columns by the hundred.  Against the definitions in 64 bits, with the checks of test_gpu_rmsnorm.py."""
import pytest
import torch

import test_gpu_rmsnorm as norm

pytestmark = pytest.mark.gpu

LARGE = [(33000, 512), (17000, 1000), (8300, 2048), (4100, 4104)]


@pytest.mark.parametrize("rows,D", [(700, 4104), (333, 8192), *LARGE])
def test_forward_without_a_residual(rows, D):
    x, _, gamma = norm.inputs(rows, D, rows + D)
    _, y, q, scales = norm.forward(x, None, gamma)
    v = norm.normalised(x, gamma)
    norm.near(y, v, v.abs() * (2.0 ** -8 + norm.FP32), "y")
    norm.check_codes(q, scales, v)


@pytest.mark.parametrize("rows,D", [(700, 4104), (333, 8192), *LARGE])
def test_forward(rows, D):
    norm.test_forward(rows, D)


@pytest.mark.parametrize("rows,D", [(700, 4104), (333, 8192), *LARGE])
def test_backward(rows, D):
    norm.test_backward(rows, D)


