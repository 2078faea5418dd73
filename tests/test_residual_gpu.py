"""GPU parity of the GEMM with a residual in its epilogue, act(a @ b.T + bias) + residual, against the oracle's fp32 sums."""
import numpy as np
import pytest
import torch

from helpers import assert_bit_exact

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sub(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nvfp4_gemm_b200 import submission
    return submission


def _expected(oracle, data, bias, activation, residual):
    """The sums are exact in fp32 (scales are powers of two), so the rounding is the only one: bit for bit."""
    a, b, sfa, sfb = oracle.tensors_to_numpy(data)
    z = oracle.ref_gemm_f32(a, b, sfa, sfb).astype(np.float32)
    if bias is not None:
        z = z + bias.cpu().numpy().astype(np.float32)[None, :, None]
    if activation == "relu":
        z = np.maximum(z, np.float32(0))
    with np.errstate(over="ignore"):
        return (z + residual.cpu().numpy().astype(np.float32)).astype(np.float16)


def _inputs(shape, seed):
    from nvfp4_gemm_b200.inputs import generate_input
    m, n, k, l = shape
    data = generate_input(m, n, k, l, seed)
    g = torch.Generator().manual_seed(seed)
    bias = (torch.randn(n, generator=g) * 64).half().cuda()
    residual = (torch.randn((l, m, n), generator=g) * 200).half().cuda().permute(1, 2, 0)
    return data, bias, residual


# CTA-pair 256- and 128-wide tiles, one-CTA tiles of both widths, shared tiles, cluster split-K, the decode kernels of 32, 64 and
# 128 tokens with their splits, one row, ragged rows, batches
CASES = [
    ((512, 1024, 1024, 1), dict()),
    ((300, 768, 1536, 2), dict()),
    ((384, 640, 2048, 1), dict()),
    ((256, 512, 1024, 1), dict(cta_group=1, tile_n=256)),
    ((640, 512, 2048, 1), dict(grid=4)),
    ((128, 512, 4096, 1), dict(split_k=1, grid=6)),
    ((100, 256, 2048, 1), dict(split_k=2)),
    ((1, 512, 512, 1), dict()),
    ((17, 7168, 2048, 1), dict()),
    ((17, 512, 16384, 1), dict()),
    ((33, 2048, 4096, 2), dict()),
    ((50, 20480, 256, 1), dict()),
    ((100, 1024, 4096, 1), dict()),
    ((256, 1536, 4096, 1), dict()),
]


@pytest.mark.parametrize("activation,with_bias", [("none", False), ("relu", True)])
@pytest.mark.parametrize("shape,kw", CASES)
def test_residual_fp16_bit_exact(sub, oracle, shape, kw, activation, with_bias):
    data, bias, residual = _inputs(shape, 31)
    bias = bias if with_bias else None
    data[6].view(torch.int16).fill_(0x7fff)
    exp = _expected(oracle, data, bias, activation, residual)
    out = sub.gemm_epilogue(data, bias=bias, activation=activation, residual=residual, **kw)
    sub.check_status()
    assert_bit_exact(out, exp, what=f"{shape} {activation} {sub.last_kernel()}")
    # in place: c is the residual
    data[6].copy_(residual)
    sub.gemm_epilogue(data, bias=bias, activation=activation, residual=data[6], **kw)
    sub.check_status()
    assert_bit_exact(data[6], exp, what=f"in place {shape}")


@pytest.mark.parametrize("shape,kw", CASES)
def test_requantised_sum_is_the_quantised_fp16_sum(sub, oracle, shape, kw):
    data, bias, residual = _inputs(shape, 32)
    exp = _expected(oracle, data, bias, "none", residual)
    packed, sf, sf_perm = sub.gemm_epilogue(data[:6] + (None,), bias=bias, nvfp4_out=True, residual=residual, **kw)
    sub.check_status()
    exp_packed, exp_sf = oracle.ref_requantize(exp)
    assert np.array_equal(sf.view(torch.uint8).cpu().numpy(), exp_sf)
    assert np.array_equal(packed.view(torch.uint8).cpu().numpy(), exp_packed)
    flat = torch.as_strided(sf_perm.view(torch.uint8), (sf_perm.numel(),), (1,)).cpu().numpy()
    assert np.array_equal(flat, oracle.permute_sf(exp_sf).reshape(-1))


@pytest.mark.parametrize("shape", [(40, 512, 512, 2), (300, 512, 512, 2)])
def test_strided_and_repeated_residuals(sub, oracle, shape):
    m, n, k, l = shape
    data, _, residual = _inputs(shape, 33)
    wide = torch.zeros((l, m, n + 64), dtype=torch.float16, device="cuda").permute(1, 2, 0)[:, 8:8 + n]
    wide.copy_(residual)
    exp = _expected(oracle, data, None, "none", residual)
    assert_bit_exact(sub.gemm_epilogue(data, residual=wide), exp, what="strided")
    one = residual[:1, :, :1].expand(m, n, l)
    assert_bit_exact(sub.gemm_epilogue(data, residual=one), _expected(oracle, data, None, "none", one), what="one row for all")


def test_infinities_and_nan_of_the_residual_pass_through(sub):
    data, _, residual = _inputs((20, 256, 256, 1), 34)
    residual = residual.clone()
    residual[3, 5, 0], residual[4, 6, 0], residual[5, 7, 0] = float("inf"), float("-inf"), float("nan")
    out = sub.gemm_epilogue(data, residual=residual)
    assert out[3, 5, 0] == float("inf") and out[4, 6, 0] == float("-inf") and torch.isnan(out[5, 7, 0])
    assert int((~torch.isfinite(out)).sum()) == 3


def test_residual_refusals(sub, lib):
    from nvfp4_gemm_b200 import _lib
    data, _, residual = _inputs((20, 256, 256, 1), 35)
    for bad, text in ((residual.float(), "fp16"), (residual[:10], "fp16"), (residual[:, :, 0], "fp16"), (residual.cpu(), "device")):
        with pytest.raises(ValueError, match=text):
            sub.gemm_epilogue(data, residual=bad)
    shifted = torch.zeros((20, 264), dtype=torch.float16, device="cuda")[:, 4:260].unsqueeze(2)
    with pytest.raises(_lib.Nvfp4Error, match="16-byte aligned"):
        sub.gemm_epilogue(data, residual=shifted)


def test_a_product_with_residual_that_gives_up_reports_it(sub, lib, oracle):
    """With a limit of a nanosecond waits run out while operands, and the residual's tile, are still on their way."""
    from nvfp4_gemm_b200 import _lib
    from nvfp4_gemm_b200.inputs import FP4_DTYPE, SF_DTYPE
    m, n, k = 256, 256, 1 << 22
    codes = torch.full((1, m, k // 2), 0x02, dtype=torch.uint8, device="cuda").permute(1, 2, 0).view(FP4_DTYPE)        # 1 and 0 in turn
    atoms = torch.full((1, 2, k // 64, 32, 4, 4), 0x08, dtype=torch.uint8, device="cuda").permute(3, 4, 1, 5, 2, 0).view(SF_DTYPE)   # 2^-6
    c = torch.empty((1, m, n), dtype=torch.float16, device="cuda").permute(1, 2, 0)
    data = (codes, codes, None, None, atoms, atoms, c)
    small, bias, residual = _inputs((300, 512, 512, 1), 36)
    exp = _expected(oracle, small, bias, "none", residual)
    one = torch.ones_like(c)
    kw = dict(cta_group=2, tile_n=256, grid=2, split_k=1)
    torch.cuda.synchronize()
    for _ in range(2):
        prev = lib.nvfp4_set_wait_timeout_ns(1)
        try:
            sub.gemm_epilogue(data, residual=one, **kw)
        finally:
            lib.nvfp4_set_wait_timeout_ns(prev)
        assert sub.last_kernel() == "gemm_2cta_n256_s4_residual_tmastore"
        with pytest.raises(_lib.Nvfp4Error) as e:
            sub.check_status()
        assert e.value.code == _lib.NVFP4_ERR_DEVICE_TIMEOUT
        out = sub.gemm_epilogue(small, bias=bias, residual=residual)
        sub.check_status()
        assert_bit_exact(out, exp, what="after a launch that gave up")
    sub.gemm_epilogue(data, residual=one, **kw)
    sub.check_status()
    assert torch.equal(c, torch.full_like(c, k // 2 * 2.0 ** -12 + 1))       # 512 + 1: exact
