"""Forms of the experts' operators and of the product with a residual that callers can choose: gated products with a bias, re-quantised ones with
everything, SiLU ahead of a residual, strides of every operand, and the tables of long prompts."""
import math

import numpy as np
import pytest
import torch

import experts_ref as ref
from test_experts_gpu import PRODUCTS, _check_product, _gen, _operand_values, _rows, _tile_tokens, _weights
from test_residual_gpu import CASES, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nvfp4_gemm_b200 import experts
    return experts


@pytest.fixture(autouse=True)
def _no_timeouts(request):
    yield
    if torch.cuda.is_available():
        from nvfp4_gemm_b200 import submission
        submission.check_status()


# ------------------------------------------------------------------------------------------ long prompts
def _check_tables(lib, r, ids, num_experts):
    """Rows, offsets, tile table and the rows of the scales (the last words of the plan), all against the definition."""
    tokens, top_k = ids.shape
    rows, offsets = ref.order(ids, num_experts)
    assert torch.equal(r.rows.cpu(), rows) and torch.equal(r.offsets.cpu(), offsets)
    tile = _tile_tokens(lib, tokens, top_k, num_experts)
    exp = [[e, a, min(tile, int(offsets[e + 1]) - a), 0] for e in range(num_experts) for a in range(int(offsets[e]), int(offsets[e + 1]), tile)]
    plan = r.plan.cpu()
    assert int(plan[0]) == len(exp) and plan[4:4 + 4 * len(exp)].view(-1, 4).tolist() == exp
    where = torch.cat([ref.sf_rows(offsets, tile), torch.tensor([-1])])          # row -1: none
    assert torch.equal(plan[-tokens * top_k:].view(tokens, top_k).long(), where[rows.long()])


# one chunk, one chunk a CTA, two chunks a CTA with a whole and a partial last pair of chunks; tiles of 32 and of 256 rows
@pytest.mark.parametrize("tokens,top_k,experts", [(100, 4, 8), (1000, 3, 64), (3840, 2, 16), (3841, 2, 16), (3900, 3, 16), (4000, 9, 300), (4100, 1, 1024), (5000, 8, 256), (8192, 8, 32)])
def test_tables_of_long_prompts(ex, lib, tokens, top_k, experts):
    ids = torch.randint(-1, experts + 1, (tokens, top_k), generator=_gen(tokens), dtype=torch.int32)
    _check_tables(lib, ex.plan(ids.cuda(), experts), ids, experts)
    ids = torch.where(ids % 3 == 0, torch.full_like(ids, experts // 2), ids)           # one expert has a third of all
    _check_tables(lib, ex.plan(ids.cuda(), experts), ids, experts)


@pytest.mark.parametrize("tokens,top_k,experts", [(4100, 2, 40), (5000, 4, 256)])
def test_tables_of_a_routed_prompt(ex, lib, tokens, top_k, experts):
    logits = torch.randn((tokens, experts), generator=_gen(experts))
    r = ex.route(logits.cuda(), top_k)
    assert torch.equal(r.experts.cpu().long(), logits.topk(top_k, 1).indices)
    _check_tables(lib, r, r.experts.cpu(), experts)


@pytest.mark.parametrize("tokens,top_k,experts", [(4100, 2, 40), (4200, 4, 1024)])       # 256 and 32 rows at a time
def test_quantiser_and_product_of_a_long_prompt(ex, lib, oracle, tokens, top_k, experts):
    n, k = 128, 256
    g = _gen(experts)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=g, dtype=torch.int32)
    ids[torch.rand((tokens, top_k), generator=g) < 0.2] = 7                # a long expert
    x = torch.randn((tokens, k), generator=g).bfloat16()
    r = ex.plan(ids.cuda(), experts)
    rows = ex.quantize_routed(x.cuda(), r)
    a = _operand_values(lib, r, rows, tokens, top_k, experts, k)
    packed, sf = oracle.quantize_rows(x.float().numpy())
    exp = ref.values(torch.from_numpy(packed), torch.from_numpy(sf))
    used = r.rows.cpu() >= 0
    token = torch.empty(int(r.offsets[-1]), dtype=torch.long)
    token[r.rows.cpu()[used].long()] = torch.arange(tokens).unsqueeze(1).expand(tokens, top_k)[used]
    assert torch.equal(a.cpu(), exp[token])
    w, w_sf, wv = _weights(experts, n, k, 3)
    y = ex.expert_gemm(rows, r, w, w_sf)
    z, size = ref.expert_product(a, r.offsets.cpu(), wv, None, None)
    _check_product(y[:int(r.offsets[-1])], z, size, "none", 1.0, k)


# ------------------------------------------------------------------------------------------ grouped product
def _scale_and_bias(experts, n, k):
    g = torch.Generator(device="cuda").manual_seed(1)
    return (torch.rand(experts, generator=g, device="cuda") + 0.5) / (4 * math.sqrt(k)), torch.randn((experts, n), generator=g, device="cuda").half()


@pytest.mark.parametrize("tokens,top_k,experts,n,k", PRODUCTS)
def test_gated_product_with_a_bias(ex, lib, tokens, top_k, experts, n, k):
    r, rows, a = _rows(ex, lib, tokens, top_k, experts, k, tokens + n, skew=tokens > 200)
    w, w_sf, wv = _weights(experts, n, k, n + k)
    al, b = _scale_and_bias(experts, n, k)
    y = ex.expert_gemm(rows, r, w, w_sf, alpha=al, bias=b, activation="swiglu", out_scale=0.75)
    z, size = ref.expert_product(a, r.offsets.cpu(), wv, al, b)
    _check_product(y[:int(r.offsets[-1])], z, size, "swiglu", 0.75, k)


@pytest.mark.parametrize("activation,out_scale", [("none", 3.0), ("relu", 1.0), ("silu", 2.0), ("swiglu", 4.0)])
@pytest.mark.parametrize("tokens,top_k,experts,n,k", PRODUCTS)
def test_requantised_product_with_scale_bias_and_activation(ex, lib, oracle, tokens, top_k, experts, n, k, activation, out_scale):
    r, rows, _ = _rows(ex, lib, tokens, top_k, experts, k, tokens + k, skew=tokens > 200)
    w, w_sf, _ = _weights(experts, n, k, n)
    al, b = _scale_and_bias(experts, n, k)
    y = ex.expert_gemm(rows, r, w, w_sf, alpha=al, bias=b, activation=activation, out_scale=out_scale)
    q = ex.expert_gemm(rows, r, w, w_sf, alpha=al, bias=b, activation=activation, out_scale=out_scale, nvfp4_out=True)
    used, cols = int(r.offsets[-1]), y.shape[1]
    exp_packed, exp_sf = oracle.quantize_rows(y[:used].float().cpu().numpy())
    assert np.array_equal(q.packed.view(torch.uint8)[:used].cpu().numpy(), exp_packed)
    where = ref.sf_rows(r.offsets.cpu(), _tile_tokens(lib, tokens, top_k, experts))
    assert np.array_equal(ref.scales_of(q.sf, where, cols).cpu().numpy(), exp_sf)


@pytest.mark.parametrize("tokens", [30, 300])
def test_strided_rows_and_bias_of_a_product(ex, lib, tokens):
    top_k, experts, n, k = 2, 4, 256, 512
    r, rows, _ = _rows(ex, lib, tokens, top_k, experts, k, 9)
    w, w_sf, _ = _weights(experts, n, k, 4)
    _, bias = _scale_and_bias(experts, n, k)
    exp = ex.expert_gemm(rows, r, w, w_sf, bias=bias)
    wide = torch.randint(0, 256, (tokens * top_k, k // 2 + 64), dtype=torch.uint8, device="cuda")
    wide[:, 16:16 + k // 2] = rows.packed.view(torch.uint8)
    wide_bias = torch.full((experts, n + 24), 100.0, dtype=torch.float16, device="cuda")
    wide_bias[:, 3:3 + n] = bias
    tall = torch.zeros((2 * n, k // 2, experts), dtype=torch.uint8, device="cuda").permute(2, 0, 1).contiguous().permute(1, 2, 0)      # every other row: the weights
    tall[::2] = w.view(torch.uint8)
    y = ex.expert_gemm((wide[:, 16:16 + k // 2], rows.sf), r, tall[::2], w_sf, bias=wide_bias[:, 3:3 + n])
    used = int(r.offsets[-1])
    assert torch.equal(y[:used], exp[:used])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_strided_and_repeated_rows_of_the_quantiser(ex, dtype):
    tokens, k, top_k, experts = 50, 320, 3, 6
    g = _gen(5)
    r = ex.plan(torch.randint(-1, experts, (tokens, top_k), generator=g, dtype=torch.int32).cuda(), experts)
    used = int(r.offsets[-1])
    wide = torch.randn((tokens, k + 40), generator=g).to(dtype).cuda()
    for x in (wide[:, 8:8 + k], wide[:, 16:16 + k], wide[3:4, :k].expand(tokens, k)):
        got, exp = ex.quantize_routed(x, r), ex.quantize_routed(x.contiguous(), r)
        assert torch.equal(got.packed.view(torch.uint8)[:used], exp.packed.view(torch.uint8)[:used])
        where = r.plan[-tokens * top_k:]
        where = where[where >= 0].long().cpu()
        assert torch.equal(ref.scales_of(got.sf, where, k), ref.scales_of(exp.sf, where, k))


# --------------------------------------------------------------------------------------------- combination
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("top_k", [1, 3, 8, 11])
def test_strided_and_repeated_operands_of_the_combination(ex, dtype, top_k):
    tokens, n = 70, 264
    g = torch.Generator(device="cuda").manual_seed(top_k)
    y = torch.randn((tokens * top_k, n + 32), generator=g, device="cuda").half()[:, 16:16 + n]
    x = torch.randn((tokens, n + 16), generator=g, device="cuda").to(dtype)[:, 8:8 + n]
    rows = torch.randint(-1, tokens * top_k, (tokens, top_k), generator=g, device="cuda", dtype=torch.int32)
    weights = torch.rand((tokens, top_k), generator=g, device="cuda")
    exp = ex.combine(y.contiguous(), rows, weights, residual=x.contiguous())
    assert exp.dtype == dtype and torch.equal(ex.combine(y, rows, weights, residual=x), exp)
    wide = torch.full((tokens, n + 48), 3.0, dtype=dtype, device="cuda")
    out = ex.combine(y, rows, weights, residual=x, out=wide[:, 24:24 + n])
    assert torch.equal(wide[:, 24:24 + n], exp) and out.data_ptr() == wide[:, 24:].data_ptr()
    assert torch.all(wide[:, :24] == 3.0) and torch.all(wide[:, 24 + n:] == 3.0)
    wide[:, 24:24 + n] = x                                              # in place, strided
    ex.combine(y, rows, weights, residual=wide[:, 24:24 + n], out=wide[:, 24:24 + n])
    assert torch.equal(wide[:, 24:24 + n], exp)
    one = x[5:6]
    assert torch.equal(ex.combine(y, rows, weights, residual=one.expand(tokens, n)), ex.combine(y, rows, weights, residual=one.repeat(tokens, 1)))
    assert torch.equal(ex.combine(y[:1].expand(tokens * top_k, n), rows, weights), ex.combine(y[:1].repeat(tokens * top_k, 1), rows, weights))


def test_a_single_expert_and_a_single_choice(ex):
    for kw in (dict(), dict(scoring="sigmoid", renormalize=False), dict(bias=torch.ones(1, device="cuda")), dict(scoring="sigmoid", bias=torch.ones(1, device="cuda"))):
        r = ex.route(torch.tensor([[0.0], [-math.inf], [5.0]], device="cuda"), 1, **kw)
        assert r.experts.tolist() == [[0], [-1], [0]] and r.rows.tolist() == [[0], [-1], [1]] and r.offsets.tolist() == [0, 2]
        exp = [0.5, 0.0, 1 / (1 + math.exp(-5.0))] if kw.get("renormalize") is False else [1.0, 0.0, 1.0]
        assert r.weights.view(-1).tolist() == pytest.approx(exp, rel=2.0 ** -19)


# ----------------------------------------------------------------------------------- product with a residual
@pytest.mark.parametrize("nvfp4_out", [False, True])
@pytest.mark.parametrize("shape,kw", CASES)
def test_silu_ahead_of_a_residual(ex, oracle, shape, kw, nvfp4_out):
    """The sums are exact in 32 bits.  Exponential, sum and quotient are within (9 + 2.35 |z|) * 2^-24 of the SiLU, which is below 2^-16 of
    it wherever it is not below 2^-126; then one addition in 32 bits and the rounding to fp16."""
    from nvfp4_gemm_b200 import submission
    data, bias, residual = _inputs(shape, 37)
    a, b, sfa, sfb = oracle.tensors_to_numpy(data)
    z = oracle.ref_gemm_f32(a, b, sfa, sfb).astype(np.float64) + bias.cpu().numpy().astype(np.float64)[None, :, None]
    with np.errstate(over="ignore"):
        silu = z / (1 + np.exp(-z))
    exp = silu + residual.cpu().numpy().astype(np.float64)
    if nvfp4_out:
        c = submission.gemm_epilogue(data, bias=bias, activation="silu", residual=residual, **kw)
        packed, sf, sf_perm = submission.gemm_epilogue(data[:6] + (None,), bias=bias, activation="silu", nvfp4_out=True, residual=residual, **kw)
        exp_packed, exp_sf = oracle.ref_requantize(c.cpu().numpy())
        # the two forms may run in kernels whose sums of a shared tile differ in nothing (they are exact), and SiLU is the same instructions
        assert np.array_equal(sf.view(torch.uint8).cpu().numpy(), exp_sf) and np.array_equal(packed.view(torch.uint8).cpu().numpy(), exp_packed)
        return
    out = submission.gemm_epilogue(data, bias=bias, activation="silu", residual=residual, **kw).cpu().numpy().astype(np.float64)
    err = 2.0 ** -16 * np.abs(silu) + 2.0 ** -24 * np.abs(exp) + 2.0 ** -125
    tol = err + 2.0 ** -11 * (np.abs(exp) + err) + 2.0 ** -25
    over = np.abs(exp) >= 65504
    bad = (np.abs(out - exp) > tol) & ~over
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), submission.last_kernel())
    assert np.all(np.abs(out[over]) >= 65504 * (1 - 2.0 ** -10))
