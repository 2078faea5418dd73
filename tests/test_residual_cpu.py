"""What the GEMM with a residual refuses, before any GPU is touched."""
import pytest

from nvfp4_gemm_b200 import _lib
from nvfp4_gemm_b200.inputs import generate_input
from nvfp4_gemm_b200.submission import make_problem

A = 0x10000          # an aligned address that nothing reads: every call below is refused on the host


@pytest.mark.parametrize("ptr,row,batch,text", [
    (None, 256, 0, "residual must be"), (A + 8, 256, 0, "residual must be"), (A, 250, 0, "multiples of 8"), (A, -256, 0, "multiples of 8"),
    (A, 256, 12, "multiples of 8"), (A, 256, -8, "multiples of 8"),
])
def test_residual_refusals(lib, ptr, row, batch, text):
    data = generate_input(128, 256, 512, 2, 1, device="cpu")
    rc = lib.nvfp4_gemm_residual(make_problem(data), None, None, ptr, row, batch, None)
    assert rc == _lib.NVFP4_ERR_INVALID_ARGUMENT and text in lib.nvfp4_last_error().decode()


def test_the_gemms_own_refusals_come_first(lib):
    data = generate_input(128, 256, 512, 1, 1, device="cpu")
    p = make_problem(data)
    p.k = 300
    assert lib.nvfp4_gemm_residual(p, None, None, A, 256, 0, None) == _lib.NVFP4_ERR_INVALID_ARGUMENT
    assert "multiple of 256" in lib.nvfp4_last_error().decode()
    epi = _lib.Epilogue()
    epi.activation = 7
    assert lib.nvfp4_gemm_residual(make_problem(data), None, epi, A, 256, 0, None) == _lib.NVFP4_ERR_INVALID_ARGUMENT
