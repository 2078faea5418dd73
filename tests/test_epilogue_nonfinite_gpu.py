"""NaN and infinities through the GEMM's extended epilogue, with and without a residual: an activation keeps a NaN."""
import math

import pytest
import torch

from helpers import assert_bit_exact
from test_residual_gpu import CASES, _expected, _inputs

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def sub(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nvfp4_gemm_b200 import submission
    return submission


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("shape,kw", CASES)
def test_relu_keeps_nan(sub, oracle, shape, kw, with_residual):
    data, bias, residual = _inputs(shape, 41)
    n = shape[1]
    bias[3], bias[n // 2 + 1], bias[n - 1], bias[n // 2] = NAN, NAN, INF, -INF
    out = sub.gemm_epilogue(data, bias=bias, activation="relu", residual=residual if with_residual else None, **kw).clone()
    sub.check_status()
    exp = _expected(oracle, data, bias, "relu", residual if with_residual else torch.zeros_like(residual))
    nan = torch.zeros(n, dtype=torch.bool)
    nan[3] = nan[n // 2 + 1] = True
    got = out.cpu()
    assert torch.equal(torch.isnan(got), nan.view(1, n, 1).expand(got.shape)), sub.last_kernel()
    keep = ~nan
    assert_bit_exact(got[:, keep], exp[:, keep.numpy()], what=f"{shape} {sub.last_kernel()}")
