"""What the native module refuses of the epilogue's tensors.  Tensors that say they are on a device which no machine has stand in for those
of a GPU: what is refused is refused before that device is looked for."""
import subprocess
import sys
from pathlib import Path

import pytest

_SETUP = """
import torch
from nvfp4_gemm_b200 import submission

class Elsewhere(torch.Tensor):
    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(func)

def tensor(*shape, dtype=torch.uint8, strides=None, device="cuda:63"):
    if strides is None:
        strides = [1] * len(shape)
        order = [1, 0, *range(2, len(shape))][:len(shape)] if len(shape) > 1 else [0]
        step = 1
        for i in order:
            strides[i], step = step, step * shape[i]
    return torch.Tensor._make_wrapper_subclass(Elsewhere, shape, strides=strides, dtype=dtype, device=device)

data = (tensor(128, 128, 1), tensor(256, 128, 1), None, None, None, None, tensor(128, 256, 1, dtype=torch.float16))

def call(**kw):
    try:
        submission.gemm_epilogue(data, **kw)
    except Exception as e:
        print(type(e).__name__, e)
"""


def _run(lib, text):
    r = subprocess.run([sys.executable, "-c", _SETUP + text], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout.strip()


@pytest.mark.parametrize("residual", ["None", "tensor(128, 256, 1, dtype=torch.float16)"])
def test_a_bias_of_another_device_is_refused(lib, residual):
    """Its address would be the kernel's to read."""
    for bias in ("torch.zeros(256, dtype=torch.float16)", "tensor(256, dtype=torch.float16, device='cuda:62')"):
        assert _run(lib, f"call(bias={bias}, residual={residual})") == "ValueError bias must be on the device of a"
    # one of the same device goes on to the device, which is not there
    assert _run(lib, f"call(bias=tensor(256, dtype=torch.float16), residual={residual})").split()[0] in ("RuntimeError", "AcceleratorError")


@pytest.mark.parametrize("place,bad,text", [
    (0, "tensor(127, 128)", "hold"), (1, "tensor(128, 15)", "hold"), (2, "tensor(128, 15)", "hold"),
    (0, "tensor(128, 128, dtype=torch.float16)", "hold"), (1, "tensor(128, 16, strides=[32, 1])", "hold"),
    (0, "tensor(128, 128, device='cuda:62')", "device of a"), (1, "torch.zeros((128, 16), dtype=torch.uint8)", "device of a"),
])
def test_memory_that_does_not_hold_the_result_is_refused(lib, place, bad, text):
    """The kernel would write past it, or to another device's address."""
    out = ["tensor(128, 128)", "tensor(128, 16)", "tensor(128, 16)"]
    out[place] = bad
    answer = _run(lib, f"call(nvfp4_out=True, out=({', '.join(out)}))")
    assert answer.startswith("ValueError") and text in answer
