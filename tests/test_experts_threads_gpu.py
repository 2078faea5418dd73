"""The experts' operators and the dense product from several threads at once, the first calls on a device among them."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

# In a process of its own, so that the first calls of all are made side by side.
_SCRIPT = """
import threading
import torch
from nvfp4_gemm_b200 import experts as X, submission as S
from nvfp4_gemm_b200.inputs import generate_input

g = torch.Generator(device="cuda").manual_seed(1)
E, K, D, F = 8, 2, 512, 256
def weights(n, k):
    codes = torch.randint(0, 256, (E, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    sf = torch.full((E, n // 128, k // 64, 32, 4, 4), 0x38, dtype=torch.uint8, device="cuda")
    return codes.permute(1, 2, 0), sf.permute(3, 4, 1, 5, 2, 0)
up, down = weights(2 * F, D), weights(D, F)
al = torch.full((E,), 0.01, device="cuda")
tokens = (3, 300, 40, 700)
x = [torch.randn((t, D), generator=g, device="cuda").half() for t in tokens]
logits = [torch.randn((t, E), generator=g, device="cuda") for t in tokens]
dense = [generate_input(512, 512, 512, 1, i) for i in range(4)]
torch.cuda.synchronize()
got, errors, start = [[] for _ in tokens], [], threading.Barrier(len(tokens))

def work(i):
    try:
        start.wait()
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append((X.expert_layer(x[i], logits[i], up, down, K, up_alpha=al, down_alpha=al, residual=x[i]),
                               S.gemm_epilogue(dense[i], activation="relu", residual=x[i][:1, :].view(1, D, 1).expand(512, D, 1)).clone()))
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        errors.append(repr(e))

threads = [threading.Thread(target=work, args=(i,)) for i in range(len(tokens))]
[t.start() for t in threads]
[t.join() for t in threads]
assert not errors, errors
S.check_status()
for i in range(len(tokens)):
    layer = X.expert_layer(x[i], logits[i], up, down, K, up_alpha=al, down_alpha=al, residual=x[i])
    product = S.gemm_epilogue(dense[i], activation="relu", residual=x[i][:1, :].view(1, D, 1).expand(512, D, 1))
    assert all(torch.equal(a, layer) and torch.equal(b, product) for a, b in got[i]), i
S.check_status()
print("same")
"""


def test_threads_at_once(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    r = subprocess.run([sys.executable, "-c", _SCRIPT], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stdout[-500:] + r.stderr[-2000:]
