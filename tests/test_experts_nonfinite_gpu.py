"""NaN and infinities through the experts' products: what is not a number stays none, whichever activation, and nothing else changes."""
import math

import numpy as np
import pytest
import torch

import experts_ref as ref
from test_experts_gpu import _rows, _tile_tokens, _weights

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def ex(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nvfp4_gemm_b200 import experts
    return experts


def _quantised(oracle, x):
    """The quantiser's rule with what is no number: a NaN does not count towards its block's scale, and becomes +6 where the rest of
    the block is within 65504, -6 where it is not (nothing where the scale is 0); infinities saturate."""
    nan = np.isnan(x)
    rest = np.where(nan, np.float32(0), x)
    packed, sf = oracle.quantize_rows(np.clip(rest, -65504, 65504))
    far = (np.abs(rest).reshape(x.shape[0], -1, 16).max(-1) > 65504).repeat(16, -1)
    code = np.where(sf.repeat(16, -1) > 0, np.where(far, 0xF, 0x7), 0).astype(np.uint8)
    codes = np.stack([packed & 15, packed >> 4], -1).reshape(x.shape)
    codes = np.where(nan, code, codes)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8), sf


# few rows per expert (single CTAs) and many (pairs); one and several 32-row pieces
@pytest.mark.parametrize("tokens", [20, 300])
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "swiglu"])
def test_nan_and_infinities_of_alpha_and_bias(ex, lib, oracle, tokens, activation):
    top_k, experts, n, k = 2, 4, 384, 256
    r, rows, _ = _rows(ex, lib, tokens, top_k, experts, k, tokens)
    w, w_sf, _ = _weights(experts, n, k, 2)
    offsets = r.offsets.tolist()
    g = torch.Generator(device="cuda").manual_seed(3)
    alpha = torch.full((experts,), 1.0 / 64, device="cuda")
    bias = torch.randn((experts, n), generator=g, device="cuda").half()
    clean = ex.expert_gemm(rows, r, w, w_sf, alpha=alpha, bias=bias, activation=activation)
    bias[1, 5], bias[1, 70], bias[2, 200], bias[2, 209], bias[1, 383] = NAN, INF, -INF, NAN, NAN
    alpha[3] = NAN
    y = ex.expert_gemm(rows, r, w, w_sf, alpha=alpha, bias=bias, activation=activation)
    exp = clean.clone()
    if activation == "swiglu":      # 16 rows of the weights are gate and up of 8 columns; these are all of gates and of an up
        at = lambda row: row // 16 * 8 + row % 8                      # noqa: E731
        exp[offsets[1]:offsets[2], [at(5), at(383)]] = NAN            # a gate, an up
        exp[offsets[2]:offsets[3], [at(200), at(209)]] = NAN          # silu(z_gate) * -inf is -+inf, see below; a gate
    else:
        exp[offsets[1]:offsets[2], [5, 383]] = NAN
        exp[offsets[2]:offsets[3], 209] = NAN
        exp[offsets[1]:offsets[2], 70] = INF
        exp[offsets[2]:offsets[3], 200] = {"none": -INF, "relu": 0.0, "silu": NAN}[activation]     # z / (1 + exp(-z)) of -inf
    exp[offsets[3]:offsets[4]] = NAN
    if activation == "swiglu":
        # an infinite gate or up: infinite with the sign of the other factor (70: a gate, 200: an up)
        for e, row in ((1, 70), (2, 200)):
            got = y[offsets[e]:offsets[e + 1], at(row)]
            assert torch.all(torch.isinf(got))
            exp[offsets[e]:offsets[e + 1], at(row)] = got
    used = offsets[-1]
    assert torch.equal(torch.isnan(y[:used]), torch.isnan(exp[:used])), (torch.isnan(y[:used]) != torch.isnan(exp[:used])).nonzero()[:4].tolist()
    assert torch.equal(torch.nan_to_num(y[:used], nan=0.0), torch.nan_to_num(exp[:used], nan=0.0))
    # the re-quantised form is the quantiser's of these values
    q = ex.expert_gemm(rows, r, w, w_sf, alpha=alpha, bias=bias, activation=activation, nvfp4_out=True)
    exp_packed, exp_sf = _quantised(oracle, y[:used].float().cpu().numpy())
    assert np.array_equal(q.packed.view(torch.uint8)[:used].cpu().numpy(), exp_packed)
    where = ref.sf_rows(r.offsets.cpu(), _tile_tokens(lib, tokens, top_k, experts))
    assert np.array_equal(ref.scales_of(q.sf, where, y.shape[1]).cpu().numpy(), exp_sf)


@pytest.mark.parametrize("tokens", [20, 300])
@pytest.mark.parametrize("activation", ["none", "relu", "silu"])
def test_nan_among_the_block_scales(ex, lib, tokens, activation):
    """A NaN scale of a block of weights makes its column NaN, one of a row's block the row."""
    top_k, experts, n, k = 2, 4, 256, 512
    r, rows, _ = _rows(ex, lib, tokens, top_k, experts, k, tokens + 1)
    w, w_sf, _ = _weights(experts, n, k, 2)
    offsets = r.offsets.tolist()
    exp = ex.expert_gemm(rows, r, w, w_sf, activation=activation).clone()
    row, col, block = 133, 9, 7                     # of expert 1, and the scale of k-block 7: atom 1, entry 3
    w_sf.view(torch.uint8)[row % 32, (row % 128) // 32, row // 128, block % 4, block // 4, 1] = 0x7F
    where = ref.sf_rows(r.offsets.cpu(), _tile_tokens(lib, tokens, top_k, experts))
    at = int(where[col])                            # row 9 in expert order
    atoms = rows.sf.view(torch.uint8).view(-1, k // 64, 32, 4, 4)
    atoms[at // 128, block // 4, at % 32, (at % 128) // 32, block % 4] = 0x7F
    y = ex.expert_gemm(rows, r, w, w_sf, activation=activation)
    exp[offsets[1]:offsets[2], row] = NAN
    exp[col] = NAN
    used = offsets[-1]
    assert torch.equal(torch.isnan(y[:used]), torch.isnan(exp[:used]))
    assert torch.equal(torch.nan_to_num(y[:used], nan=0.0), torch.nan_to_num(exp[:used], nan=0.0))
