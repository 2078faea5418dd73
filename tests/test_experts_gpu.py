"""GPU parity of the mixture-of-experts operators -- router and plan, routed quantiser, grouped product, combination -- against
their definitions in 64 bits (experts_ref.py) and, for what the quantiser writes, against the oracle bit for bit."""
import ctypes
import math

import numpy as np
import pytest
import torch

import experts_ref as ref

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


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


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _tile_tokens(lib, tokens, top_k, experts):
    t = ctypes.c_int32()
    assert lib.nvfp4_routing_plan(tokens, top_k, experts, ctypes.byref(t), None, None) == 0
    return t.value


# ---------------------------------------------------------------------------------------------- router
def _check_routing(lib, r, logits, top_k, num_experts, **kw):
    experts, weights = ref.route(logits, top_k, **kw)
    assert torch.equal(r.experts.cpu(), experts)
    # weights: a sum of at most 1024 exponentials in 32 bits, 32 in a row in each lane and 5 steps across lanes, each exponential within
    # 2 units of 2^-24 .. 2^-23, one rounding of the result: below 64 * 2^-24
    got = r.weights.cpu().double()
    assert torch.all((got - weights).abs() <= 2.0 ** -18 * weights.abs() + 1e-45), (got - weights).abs().max()
    rows, offsets = ref.order(experts, num_experts)
    assert torch.equal(r.rows.cpu(), rows) and torch.equal(r.offsets.cpu(), offsets)
    # the tile table: every expert's rows once, in pieces of at most tile_tokens
    tile = _tile_tokens(lib, logits.shape[0], top_k, num_experts)
    exp = [[e, a, min(tile, int(offsets[e + 1]) - a), 0] for e in range(num_experts) for a in range(int(offsets[e]), int(offsets[e + 1]), tile)]
    plan = r.plan.cpu()
    assert int(plan[0]) == len(exp) and plan[4:4 + 4 * len(exp)].view(-1, 4).tolist() == exp


ROUTERS = [
    dict(),
    dict(renormalize=False, scale=2.5),
    dict(scoring="sigmoid"),
    dict(scoring="sigmoid", bias=True, renormalize=False),
    dict(bias=True),
    dict(groups=4, top_groups=2),
    dict(scoring="sigmoid", bias=True, groups=4, top_groups=3, group_score="top2", scale=2.5),
    dict(groups=8, top_groups=4, group_score="top2"),
]


@pytest.mark.parametrize("kw", ROUTERS, ids=str)
@pytest.mark.parametrize("tokens,experts,top_k,dtype", [
    (1, 8, 1, torch.float32), (5, 8, 3, torch.bfloat16), (32, 64, 6, torch.float16), (33, 40, 4, torch.float32),
    (200, 256, 8, torch.bfloat16), (70, 384, 8, torch.float32), (40, 1024, 32, torch.float32)])
def test_router_against_its_definition(ex, lib, tokens, experts, top_k, dtype, kw):
    g = _gen(tokens + experts)
    logits = (torch.randn((tokens, experts), generator=g) * 2).to(dtype)       # bf16 and fp16: equal logits occur
    kw = dict(kw)
    if kw.get("top_groups", 1) * (experts // kw.get("groups", 1)) < top_k:
        pytest.skip("fewer experts in the groups than choices")
    if kw.get("bias"):
        kw["bias"] = torch.randn(experts, generator=g) * 0.2
    r = ex.route(logits.cuda(), top_k, **{**kw, **({"bias": kw["bias"].cuda()} if "bias" in kw else {})})
    _check_routing(lib, r, logits, top_k, experts, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(scoring="sigmoid"), dict(bias=True), dict(groups=4, top_groups=2), dict(scoring="sigmoid", bias=True, groups=4, top_groups=2, group_score="top2")], ids=str)
def test_masked_infinite_and_nan_logits(ex, lib, kw):
    experts, top_k = 16, 4
    g = _gen(7)
    x = torch.randn((10, experts), generator=g)
    x[0] = -INF                                      # nothing left
    x[1, 3:] = -INF                                  # three left of four asked for
    x[2] = NAN
    x[3, ::2] = NAN
    x[4] = torch.finfo(torch.float32).min            # masked by the type's lowest value: all alike
    x[5, 1:] = torch.finfo(torch.float32).min
    x[6, 5], x[6, 9] = INF, INF
    x[7] = 0.0
    x[7, ::2] = -0.0                                 # +0 and -0 are a tie
    x[8, 2] = 1e30
    x[9] = -1e4                                      # sigmoid: all scores 0 or tiny
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = torch.randn(experts, generator=g) * 0.2
        kw["bias"][6], kw["bias"][7] = -INF, NAN
    r = ex.route(x.cuda(), top_k, **{**kw, **({"bias": kw["bias"].cuda()} if "bias" in kw else {})})
    _check_routing(lib, r, x, top_k, experts, **kw)


def test_scores_nearer_than_their_32_bit_rounding(ex, lib):
    """Large logits whose sigmoids are one and the same fp32 number are told apart, with and without bias."""
    x = torch.linspace(17.0, 20.0, 64).flip(0).repeat(2, 1).contiguous()
    x[1] = x[1].flip(0)
    assert (torch.sigmoid(x) == 1.0).sum() > 64
    for kw in (dict(scoring="sigmoid"), dict(scoring="sigmoid", bias=torch.zeros(64))):
        r = ex.route(x.cuda(), 5, **{**kw, **({"bias": kw["bias"].cuda()} if "bias" in kw else {})})
        assert r.experts.cpu().tolist() == [[0, 1, 2, 3, 4], [63, 62, 61, 60, 59]]


def test_logits_with_a_row_stride_and_a_broadcast_row(ex, lib):
    g = _gen(3)
    wide = torch.randn((50, 100), generator=g)
    view = wide[:, 13:77]
    _check_routing(lib, ex.route(wide.cuda()[:, 13:77], 4), view, 4, 64)
    one = torch.randn((1, 32), generator=g)
    _check_routing(lib, ex.route(one.cuda().expand(40, 32), 2), one.expand(40, 32), 2, 32)


@pytest.mark.parametrize("tokens,top_k,experts", [(1, 1, 1), (3, 2, 5), (32, 8, 64), (33, 1, 7), (5000, 8, 256), (9000, 3, 16), (148 * 32 + 1, 4, 1024)])
def test_plan_of_given_choices(ex, lib, tokens, top_k, experts):
    g = _gen(tokens)
    ids = torch.randint(-1, experts + 1, (tokens, top_k), generator=g, dtype=torch.int32)      # -1 and experts: none; the same expert may be there twice
    r = ex.plan(ids.cuda(), experts)
    rows, offsets = ref.order(ids, experts)
    assert torch.equal(r.rows.cpu(), rows) and torch.equal(r.offsets.cpu(), offsets) and r.weights is None


def test_plan_where_all_tokens_want_one_expert(ex):
    ids = torch.full((3000, 2), 5, dtype=torch.int32)
    r = ex.plan(ids.cuda(), 40)
    assert torch.equal(r.rows.cpu().view(-1), torch.arange(6000, dtype=torch.int32))
    assert r.offsets.tolist() == [0] * 6 + [6000] * 35


def test_no_tokens(ex):
    r = ex.route(torch.empty((0, 64), device="cuda"), 4)
    assert r.experts.shape == (0, 4) and r.offsets.tolist() == [0] * 65
    rows = ex.quantize_routed(torch.empty((0, 256), dtype=torch.bfloat16, device="cuda"), r)
    w, sf, _ = _weights(64, 128, 256, 1)
    y = ex.expert_gemm(rows, r, w, sf)
    assert y.shape == (0, 128)
    assert ex.combine(y, r.rows, r.weights).shape == (0, 128)


# --------------------------------------------------------------------------------------- routed quantiser
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,k,top_k,experts,aligned", [(1, 64, 1, 4, True), (7, 576, 3, 5, True), (40, 1024, 2, 8, False), (300, 256, 8, 16, True)])
def test_routed_quantiser_against_the_oracle(ex, lib, oracle, dtype, tokens, k, top_k, experts, aligned):
    g = _gen(k)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=g, dtype=torch.int32)
    x = (torch.randn((tokens, k), generator=g) * torch.exp(torch.randn((tokens, 1), generator=g))).to(dtype)
    x[0, :16] = 0
    dev = torch.empty((tokens, k + 8), dtype=dtype, device="cuda")[:, 8 if not aligned else 0:][:, :k]
    dev.copy_(x)
    r = ex.plan(ids.cuda(), experts)
    packed, sf = ex.quantize_routed(dev, r)
    exp_packed, exp_sf = oracle.quantize_rows(x.float().numpy())
    rows, offsets = ref.order(ids, experts)
    n = int(offsets[-1])
    token = torch.empty(n, dtype=torch.long)
    token[rows[rows >= 0].long()] = torch.arange(tokens).repeat_interleave(top_k).view(tokens, top_k)[rows >= 0]
    assert np.array_equal(packed.view(torch.uint8)[:n].cpu().numpy(), exp_packed[token.numpy()])
    where = ref.sf_rows(offsets, _tile_tokens(lib, tokens, top_k, experts))
    assert np.array_equal(ref.scales_of(sf, where, k).cpu().numpy(), exp_sf[token.numpy()])


# ------------------------------------------------------------------------------------------ grouped product
def _weights(experts, n, k, seed):
    """4-bit weights in the operator's layout, and their float64 values [E, N, K]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (experts, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    sf = torch.randint(40, 72, (experts, n, k // 16), generator=g, device="cuda", dtype=torch.uint8)     # 0.25 .. 3.75
    from nvfp4_gemm_b200.inputs import FP4_DTYPE, SF_DTYPE, permute_scale_factors
    return codes.permute(1, 2, 0).view(FP4_DTYPE), permute_scale_factors(sf).view(SF_DTYPE), ref.values(codes, sf)


def _rows(ex, lib, tokens, top_k, experts, k, seed, skew=False):
    """A routing with some pairs that are none, its routed operand, and the operand's float64 values in expert order."""
    g = _gen(seed)
    ids = torch.randint(0, experts, (tokens, top_k), generator=g, dtype=torch.int32)
    if skew:
        ids = torch.where(torch.rand((tokens, top_k), generator=g) < 0.7, torch.full_like(ids, experts // 2), ids)
    ids[torch.rand((tokens, top_k), generator=g) < 0.1] = -1
    ids[0, 0] = experts - 1
    r = ex.plan(ids.cuda(), experts)
    x = torch.randn((tokens, k), generator=g).bfloat16().cuda()
    rows = ex.quantize_routed(x, r)
    return r, rows, _operand_values(lib, r, rows, tokens, top_k, experts, k)


def _operand_values(lib, r, rows, tokens, top_k, experts, k):
    n = int(r.offsets[-1])
    where = ref.sf_rows(r.offsets.cpu(), _tile_tokens(lib, tokens, top_k, experts))
    return ref.values(rows.packed.view(torch.uint8)[:n], ref.scales_of(rows.sf, where, k))


def _check_product(y, z, size, activation, out_scale, k):
    # the sum: K / 64 accumulations and a few more roundings, each within 2^-22 of the sum of absolute products (an fp32
    # accumulator that may truncate); silu: exponential and division within 2^-19 for |z| < 16; the fp16 result: half a step
    e = (k / 64 + 4) * 2.0 ** -22 * size
    exp = out_scale * ref.activate(z, activation)
    if activation == "swiglu":
        p, q = z.unflatten(-1, (-1, 2, 8)), e.unflatten(-1, (-1, 2, 8))
        g, u = p[..., 0, :], p[..., 1, :]
        s = g / (1 + torch.exp(-g))
        err = out_scale * (1.1 * q[..., 0, :] * u.abs() + s.abs() * q[..., 1, :] + 1.2 * q[..., 0, :] * q[..., 1, :]).flatten(-2) + 2.0 ** -18 * exp.abs()
    elif activation == "silu":
        err = out_scale * 1.1 * e + 2.0 ** -18 * exp.abs()
    else:
        err = out_scale * e
    tol = err + 2.0 ** -11 * (exp.abs() + err) + 2.0 ** -25
    bad = (y.double() - exp).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.numel(), float(((y.double() - exp).abs() / tol).max()), bad.nonzero()[:4].tolist())


# few rows per expert (single CTAs) and many (pairs); n that ends inside a pair's tile; one and several k-tiles; tiles of 1 to 256 rows and more
PRODUCTS = [
    (1, 1, 4, 128, 256), (3, 4, 8, 384, 512), (24, 2, 4, 256, 1024), (17, 8, 64, 640, 2048), (65, 1, 5, 128, 256),
    (100, 4, 8, 384, 256), (260, 2, 2, 256, 768), (700, 2, 3, 896, 512), (1024, 4, 8, 512, 2048), (64, 8, 16, 512, 7168),
]


@pytest.mark.parametrize("activation,bias,alpha,out_scale", [("none", False, False, 1.0), ("relu", True, True, 1.0), ("silu", True, True, 0.5), ("swiglu", False, True, 2.0)])
@pytest.mark.parametrize("tokens,top_k,experts,n,k", PRODUCTS)
def test_grouped_product_against_its_definition(ex, lib, tokens, top_k, experts, n, k, activation, bias, alpha, out_scale):
    r, rows, a = _rows(ex, lib, tokens, top_k, experts, k, tokens + n, skew=tokens > 200)
    w, w_sf, wv = _weights(experts, n, k, n + k)
    g = torch.Generator(device="cuda").manual_seed(1)
    # products around 0.3 * sqrt(K) each way brought to a few units
    al = (torch.rand(experts, generator=g, device="cuda") + 0.5) / (4 * math.sqrt(k)) if alpha else None
    b = torch.randn((experts, n), generator=g, device="cuda").half() if bias else None
    cols = n // 2 if activation == "swiglu" else n
    out = torch.full((tokens * top_k, cols), 7.0, dtype=torch.float16, device="cuda")
    y = ex.expert_gemm(rows, r, w, w_sf, alpha=al, bias=b, activation=activation, out_scale=out_scale, out=out)
    assert y.data_ptr() == out.data_ptr()
    z, size = ref.expert_product(a, r.offsets.cpu(), wv, al, b)
    used = int(r.offsets[-1])
    _check_product(y[:used], z, size, activation, out_scale, k)
    assert torch.all(y[used:] == 7.0)                      # rows that nobody has are left as they were


@pytest.mark.parametrize("activation", ["none", "swiglu"])
@pytest.mark.parametrize("tokens,top_k,experts,n,k", PRODUCTS)
def test_requantised_product_is_the_quantised_fp16_product(ex, lib, oracle, tokens, top_k, experts, n, k, activation):
    r, rows, _ = _rows(ex, lib, tokens, top_k, experts, k, tokens + k, skew=tokens > 200)
    w, w_sf, _ = _weights(experts, n, k, n)
    al = torch.full((experts,), 1.0 / (4 * math.sqrt(k)), device="cuda")
    y = ex.expert_gemm(rows, r, w, w_sf, alpha=al, activation=activation)
    q = ex.expert_gemm(rows, r, w, w_sf, alpha=al, activation=activation, nvfp4_out=True)
    used, cols = int(r.offsets[-1]), y.shape[1]
    exp_packed, exp_sf = oracle.quantize_rows(y[:used].float().cpu().numpy())
    assert np.array_equal(q.packed.view(torch.uint8)[:used].cpu().numpy(), exp_packed)
    where = ref.sf_rows(r.offsets.cpu(), _tile_tokens(lib, tokens, top_k, experts))
    assert np.array_equal(ref.scales_of(q.sf, where, cols).cpu().numpy(), exp_sf)


def test_out_with_a_row_stride_and_weights_with_gaps(ex, lib):
    tokens, top_k, experts, n, k = 40, 2, 4, 256, 512
    r, rows, a = _rows(ex, lib, tokens, top_k, experts, k, 9)
    w, w_sf, wv = _weights(2 * experts, n, k, 4)
    wide = torch.zeros((tokens * top_k, n + 64), dtype=torch.float16, device="cuda")
    y = ex.expert_gemm(rows, r, w[:, :, ::2], w_sf[..., ::2], out=wide[:, 32:32 + n])
    z, size = ref.expert_product(a, r.offsets.cpu(), wv[::2], None, None)
    _check_product(y[:int(r.offsets[-1])], z, size, "none", 1.0, k)
    assert int(wide[:, :32].count_nonzero()) == 0 and int(wide[:, 32 + n:].count_nonzero()) == 0


# --------------------------------------------------------------------------------------------- combination
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,top_k,n,residual", [(1, 1, 8, True), (17, 8, 7168, True), (33, 11, 264, False), (5, 32, 1024, True), (1000, 4, 640, False)])
def test_combination_against_its_definition(ex, dtype, tokens, top_k, n, residual):
    g = torch.Generator(device="cuda").manual_seed(n)
    y = torch.randn((tokens * top_k, n), generator=g, device="cuda").half()
    rows = torch.randint(-1, tokens * top_k, (tokens, top_k), generator=g, device="cuda", dtype=torch.int32)
    if tokens > 1:
        rows[1] = -1                                                   # a token that nothing is added to
        rows[0, 0] = tokens * top_k                                    # outside y
    weights = torch.randn((tokens, top_k), generator=g, device="cuda")
    x = torch.randn((tokens, n), generator=g, device="cuda").to(dtype) if residual else None
    out = ex.combine(y, rows, weights, residual=x, dtype=dtype)
    valid = (rows >= 0) & (rows < tokens * top_k)
    terms = torch.where(valid.unsqueeze(2), weights.double().unsqueeze(2) * y.double()[rows.long().clamp(0, tokens * top_k - 1)], 0.0)
    exp = terms.sum(1) + (x.double() if residual else 0.0)
    size = terms.abs().sum(1) + (x.double().abs() if residual else 0.0)
    tol = torch.finfo(dtype).eps / 2 * exp.abs() + (top_k + 2) * 2.0 ** -24 * size + 2.0 ** -25     # the rounding, k + 1 sums in 32 bits
    assert out.dtype == dtype and torch.all((out.double() - exp).abs() <= tol)
    if residual:                                                       # in place gives the same
        again = ex.combine(y, rows, weights, residual=x, out=x)
        assert again.data_ptr() == x.data_ptr() and torch.equal(x, out)


def test_combination_ignores_what_stands_in_rows_that_are_none(ex):
    y = torch.full((4, 64), NAN, dtype=torch.float16, device="cuda")
    y[1] = 2.0
    rows = torch.tensor([[1, -1], [-1, 1]], dtype=torch.int32, device="cuda")
    out = ex.combine(y, rows, torch.full((2, 2), 0.5, device="cuda"))
    assert torch.all(out == 1.0)


# ------------------------------------------------------------------------------------------------ together
def _layer_reference(oracle, x, logits, up, down, top_k, hidden_scale, up_alpha, down_alpha, residual, **router):
    """64 bits between the roundings that the operators define: codes of x, fp16 hidden values and their codes, fp16 rows."""
    experts, weights = ref.route(logits, top_k, **router)
    packed, sf = oracle.quantize_rows(x.float().cpu().numpy())
    a = ref.values(torch.from_numpy(packed), torch.from_numpy(sf)).cuda()
    out = residual.double().clone()
    slack = torch.zeros_like(out)
    for e in range(up[2].shape[0]):
        t, j = (experts == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        z = float(up_alpha[e]) * (a[t.cuda()] @ up[2][e].t())
        h = (hidden_scale * ref.activate(z, "swiglu")).half()
        packed, sf = oracle.quantize_rows(h.float().cpu().numpy())
        hq = ref.values(torch.from_numpy(packed), torch.from_numpy(sf)).cuda()
        y = (float(down_alpha[e]) * (hq @ down[2][e].t())).half().double()
        wt = weights[t, j].cuda().unsqueeze(1)
        out.index_add_(0, t.cuda(), wt * y)
        # a hidden value next to a border of its 4-bit form may fall on the other side: up to half of it, for one in a thousand
        slack.index_add_(0, t.cuda(), wt.abs() * float(down_alpha[e]) * 0.5 * (hq.abs().amax(1, keepdim=True) * down[2][e].abs().amax(1).unsqueeze(0)))
    return out, slack


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts,top_k,d,f,router", [
    (1, 8, 2, 512, 256, dict()),
    (40, 16, 4, 256, 512, dict(scoring="sigmoid", groups=4, top_groups=2, group_score="top2", scale=2.5)),
    (300, 8, 2, 512, 256, dict(renormalize=False)),
])
def test_layer_of_all_operators(ex, oracle, dtype, tokens, experts, top_k, d, f, router):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn((tokens, d), generator=g, device="cuda").to(dtype)
    logits = torch.randn((tokens, experts), generator=g, device="cuda")
    if tokens > 1:
        logits[1] = -INF                                                  # padding: the residual goes through
    up, down = _weights(experts, 2 * f, d, 3), _weights(experts, d, f, 4)
    up_alpha = torch.full((experts,), 0.25 / math.sqrt(d), device="cuda")
    down_alpha = torch.full((experts,), 0.25 / math.sqrt(f) / 4, device="cuda")
    out = ex.expert_layer(x, logits, up[:2], down[:2], top_k, up_alpha=up_alpha, down_alpha=down_alpha, hidden_scale=4.0, residual=x, **router)
    exp, slack = _layer_reference(oracle, x, logits, up, down, top_k, 4.0, up_alpha, down_alpha, x, **router)
    err = (out.double() - exp).abs()
    assert out.dtype == dtype
    if tokens > 1:
        assert torch.equal(out[1], x[1])
    # all but a few values within their rounding (half a step of the result, of the fp16 rows, of 32-bit weights); the others within one code's change
    near = torch.finfo(dtype).eps / 2 * exp.abs() + 2.0 ** -10 * (exp - x.double()).abs().clamp(min=1.0)
    assert torch.all(err <= near + slack)
    assert float((err > near).double().mean()) < 0.02


def test_layer_captured_and_replayed_with_other_inputs(ex):
    """A captured layer follows its inputs: other tokens, other choices, without a new capture; two graphs do not disturb each other."""
    g = torch.Generator(device="cuda").manual_seed(5)
    experts, top_k, d, f = 16, 4, 512, 256
    up, down = _weights(experts, 2 * f, d, 3)[:2], _weights(experts, d, f, 4)[:2]
    al = torch.full((experts,), 0.01, device="cuda")

    def layer(x, logits):
        return ex.expert_layer(x, logits, up, down, top_k, up_alpha=al, down_alpha=al, residual=x)

    graphs = []
    for tokens in (3, 150):
        x = torch.randn((tokens, d), generator=g, device="cuda").bfloat16()
        logits = torch.randn((tokens, experts), generator=g, device="cuda")
        layer(x, logits)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, logits)
        graphs.append((graph, x, logits, out))
    for _ in range(3):
        for graph, x, logits, out in graphs:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            logits.copy_(torch.randn(logits.shape, generator=g, device="cuda"))
        for graph, *_ in graphs:
            graph.replay()
        for _, x, logits, out in graphs:
            assert torch.equal(out, layer(x, logits))


def test_layers_on_two_streams_at_once(ex):
    g = torch.Generator(device="cuda").manual_seed(6)
    experts, top_k, d, f, tokens = 8, 2, 512, 256, 200
    up, down = _weights(experts, 2 * f, d, 3)[:2], _weights(experts, d, f, 4)[:2]
    al = torch.full((experts,), 0.01, device="cuda")
    x = [torch.randn((tokens, d), generator=g, device="cuda").half() for _ in range(2)]
    logits = [torch.randn((tokens, experts), generator=g, device="cuda") for _ in range(2)]
    layer = lambda i: ex.expert_layer(x[i], logits[i], up, down, top_k, up_alpha=al, down_alpha=al, residual=x[i])  # noqa: E731
    exp = [layer(0), layer(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, exp[i]) for o in got[i])


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("experts,top_k", [(16, 3), (40, 4), (256, 8), (600, 32)])
def test_equal_scores_go_to_the_lowest_experts(ex, lib, experts, top_k, bias):
    """More equal keys than lanes, equal keys across the border of what is taken, and equal groups."""
    x = torch.zeros((4, experts))
    x[1, experts // 2:] = 1.0
    x[2, ::3] = -2.0
    x[3, experts - 1] = 5.0
    kw = dict(bias=torch.zeros(experts)) if bias else dict()
    for more in (dict(), dict(groups=4, top_groups=2), dict(groups=4, top_groups=2, group_score="top2")):
        if experts % 4 or more.get("top_groups", 9) * experts // 4 < top_k:
            continue
        r = ex.route(x.cuda(), top_k, **{k: v.cuda() for k, v in kw.items()}, **more)
        _check_routing(lib, r, x, top_k, experts, **kw, **more)


def test_scores_at_the_border_of_what_32_bits_tell_apart(ex):
    """Pairs of experts whose biased scores differ by 1e-9 .. 1e-7: in either order, among the taken and at the border, the 64-bit order decides."""
    experts, top_k = 64, 4
    g = _gen(11)
    for scoring in ("sigmoid", "softmax"):
        logits = torch.randn((200, experts), generator=g)
        bias = torch.randn(experts, generator=g) * 0.1
        s = torch.softmax(logits.double(), 1) if scoring == "softmax" else torch.sigmoid(logits.double())
        # the bias of expert 1 makes its choice almost that of expert 0 in the first token, and so on: a bias per token, one call each
        for t in range(0, 200, 8):
            b = bias.double()
            order = torch.argsort(s[t] + b, descending=True)
            for a, c in ((0, 1), (top_k - 1, top_k), (2, 3)):
                b[order[c]] += (s[t] + b)[order[a]] - (s[t] + b)[order[c]]
            b32 = b.float()                                     # a rounding of 2^-25 or so: as near as it gets
            exp, _ = ref.route(logits[t:t + 1], top_k, scoring=scoring, bias=b32)
            r = ex.route(logits[t:t + 1].cuda(), top_k, scoring=scoring, bias=b32.cuda())
            assert r.experts.cpu().tolist() == exp.tolist(), (scoring, t)


def test_infinite_biases_and_padded_tokens_by_scores(ex, lib):
    """A bias of +inf takes its expert always; tokens without any expert stand among others, in the paths that compare scores."""
    g = _gen(12)
    for experts, top_k in ((64, 4), (256, 8)):
        x = torch.randn((70, experts), generator=g)
        x[::7] = -INF
        x[3, 1:] = -INF
        bias = torch.randn(experts, generator=g) * 0.1
        for b in (bias, torch.where(torch.arange(experts) % 31 == 5, torch.tensor(INF), bias)):
            for kw in (dict(scoring="sigmoid"), dict(), dict(scoring="sigmoid", groups=8, top_groups=3, group_score="top2")):
                r = ex.route(x.cuda(), top_k, bias=b.cuda(), **kw)
                _check_routing(lib, r, x, top_k, experts, bias=b, **kw)


def test_one_expert_takes_every_row(ex, lib):
    for tokens in (3, 300):
        r, rows, a = _rows(ex, lib, tokens, 1, 1, 256, tokens)
        w, w_sf, wv = _weights(1, 256, 256, 2)
        y = ex.expert_gemm(rows, r, w, w_sf)
        z, size = ref.expert_product(a, r.offsets.cpu(), wv, None, None)
        _check_product(y[:int(r.offsets[-1])], z, size, "none", 1.0, 256)


def test_gpu_side_refusals(ex, lib):
    from nvfp4_gemm_b200 import _lib
    r = ex.route(torch.randn((6, 16), device="cuda"), 2)
    rows = ex.quantize_routed(torch.randn((6, 256), device="cuda").half(), r)
    w, w_sf, _ = _weights(16, 128, 256, 1)
    with pytest.raises(ValueError, match="row per token"):
        ex.quantize_routed(torch.randn((5, 256), device="cuda").half(), r)
    with pytest.raises(ValueError, match="fp16 or bf16"):
        ex.quantize_routed(torch.randn((6, 256), device="cuda"), r)
    with pytest.raises(ValueError, match="plan does not belong"):
        ex.expert_gemm(rows, r._replace(num_experts=700), w, w_sf)
    with pytest.raises(ValueError, match="disagree"):
        ex.expert_gemm(rows, r, w[:, :64], w_sf)
    with pytest.raises(ValueError, match="512-byte atoms"):
        ex.expert_gemm(rows, r, w, w_sf[..., :8])
    with pytest.raises(ValueError, match="routed operand"):
        ex.expert_gemm((rows.packed, rows.sf[:-16]), r, w, w_sf)
    with pytest.raises(ValueError, match="alpha"):
        ex.expert_gemm(rows, r, w, w_sf, alpha=torch.ones(15, device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        ex.expert_gemm(rows, r, w, w_sf, bias=torch.ones((16, 128), device="cuda"))
    with pytest.raises(ValueError, match="no CPU fallback"):
        ex.combine(torch.zeros((12, 128), dtype=torch.float16, device="cuda"), r.rows.cpu(), r.weights)
    with pytest.raises(_lib.Nvfp4Error, match="top_k = 17 of 16"):
        ex.route(torch.randn((6, 16), device="cuda"), 17)
    with pytest.raises(_lib.Nvfp4Error, match="groups"):
        ex.route(torch.randn((6, 16), device="cuda"), 2, groups=5)
    with pytest.raises(ValueError, match="output's type"):
        ex.combine(torch.zeros((12, 128), dtype=torch.float16, device="cuda"), r.rows, r.weights, residual=torch.zeros((6, 128), device="cuda"), dtype=torch.float16)


@pytest.mark.parametrize("tokens,kernel", [(4, "expert_gemm_t32"), (64, "expert_gemm_2cta_t256")])
def test_a_product_that_gives_up_reports_it(ex, lib, tokens, kernel):
    """With a limit of a nanosecond waits run out while a long product's operands are still streaming in.  The launch ends, the host hears
    of it, and what runs next is right."""
    from nvfp4_gemm_b200 import _lib, submission
    from nvfp4_gemm_b200.inputs import FP4_DTYPE, SF_DTYPE
    n, k = 256, 1 << 23
    r = ex.plan(torch.zeros((tokens, 1), dtype=torch.int32, device="cuda"), 1)
    w = torch.full((1, n, k // 2), 0x02, dtype=torch.uint8, device="cuda").permute(1, 2, 0).view(FP4_DTYPE)              # 1 and 0 in turn
    w_sf = torch.full((1, n // 128, k // 64, 32, 4, 4), 0x08, dtype=torch.uint8, device="cuda").permute(3, 4, 1, 5, 2, 0).view(SF_DTYPE)   # 2^-6
    sf_rows = ctypes.c_int64()
    assert lib.nvfp4_routing_plan(tokens, 1, 1, None, None, ctypes.byref(sf_rows)) == 0
    rows = ex.RoutedRows(torch.full((tokens, k // 2), 0x02, dtype=torch.uint8, device="cuda"),
                         torch.full((sf_rows.value * (k // 16),), 0x08, dtype=torch.uint8, device="cuda"))
    r2, small, a = _rows(ex, lib, 40, 2, 4, 512, 3)
    w2, w2_sf, w2v = _weights(4, 256, 512, 3)
    z, size = ref.expert_product(a, r2.offsets.cpu(), w2v, None, None)
    torch.cuda.synchronize()
    for _ in range(2):
        prev = lib.nvfp4_set_wait_timeout_ns(1)
        try:
            ex.expert_gemm(rows, r, w, w_sf)
        finally:
            lib.nvfp4_set_wait_timeout_ns(prev)
        assert submission.last_kernel() == kernel
        with pytest.raises(_lib.Nvfp4Error) as e:
            submission.check_status()
        assert e.value.code == _lib.NVFP4_ERR_DEVICE_TIMEOUT
        y = ex.expert_gemm(small, r2, w2, w2_sf)
        submission.check_status()
        _check_product(y[:int(r2.offsets[-1])], z, size, "none", 1.0, 512)
    y = ex.expert_gemm(rows, r, w, w_sf, alpha=torch.full((1,), 2.0 ** -4, device="cuda"))
    submission.check_status()
    assert torch.equal(y, torch.full_like(y, k // 2 * 2.0 ** -16))      # exact


@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(256, 8, 1, 8), (256, 8, 2, 8), (384, 8, 2, 8), (512, 8, 1, 8), (512, 32, 3, 32), (64, 16, 2, 7), (1024, 4, 1, 32)])
@pytest.mark.parametrize("kw", [dict(), dict(scoring="sigmoid", bias=True), dict(bias=True, group_score="top2")], ids=str)
def test_choices_from_few_groups(ex, lib, experts, groups, top_groups, top_k, kw):
    """What is left are the experts of a few lanes: fewer lanes than choices, and up to many more experts than lanes."""
    g = _gen(experts + top_k)
    x = torch.randn((40, experts), generator=g)
    x[5, ::2] = -INF
    x[6] = -INF
    x[6, 3] = 0.0
    kw = dict(kw, groups=groups, top_groups=top_groups)
    if kw.get("bias"):
        kw["bias"] = torch.randn(experts, generator=g) * 0.2
    if top_groups * (experts // groups) < top_k:
        pytest.skip("fewer experts in the groups than choices")
    r = ex.route(x.cuda(), top_k, **{**kw, **({"bias": kw["bias"].cuda()} if "bias" in kw else {})})
    _check_routing(lib, r, x, top_k, experts, **kw)


@pytest.mark.parametrize("experts,top_k", [(64, 24), (64, 32), (256, 20), (256, 31), (256, 32), (384, 28), (1024, 32)])
@pytest.mark.parametrize("kw", [dict(), dict(scoring="sigmoid", bias=True), dict(bias=True, groups=4, top_groups=3, group_score="top2")], ids=str)
def test_nearly_as_many_choices_as_lanes(ex, lib, experts, top_k, kw):
    g = _gen(experts + top_k)
    x = torch.randn((70, experts), generator=g)
    x[3] = x[3].bfloat16()           # ties
    x[4, 40:] = -INF
    x[5] = 0.25                      # all alike
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = torch.randn(experts, generator=g) * 0.2
    r = ex.route(x.cuda(), top_k, **{**kw, **({"bias": kw["bias"].cuda()} if "bias" in kw else {})})
    _check_routing(lib, r, x, top_k, experts, **kw)


@pytest.mark.parametrize("size", [1.0, 64.0, 4096.0])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_biases_that_outweigh_the_scores(ex, lib, size, scoring):
    """Choices whose 32-bit sums show little or nothing of the scores that tell them apart, those of the groups among them."""
    g = _gen(5)
    x = torch.randn((300, 256), generator=g)
    bias = torch.full((256,), size)
    bias[::7] += size / 64
    kw = dict(scoring=scoring, groups=8, top_groups=3, group_score="top2")
    r = ex.route(x.cuda(), 8, bias=bias.cuda(), **kw)
    _check_routing(lib, r, x, 8, 256, bias=bias, **kw)


@pytest.mark.parametrize("tokens,top_k,experts", [(176, 8, 32), (177, 8, 32), (352, 4, 128), (128, 8, 129), (256, 5, 128), (257, 5, 128), (161, 8, 64), (3900, 3, 16), (4000, 9, 300)])
def test_plans_about_the_borders_of_one_chunk_and_of_two_chunks_a_cta(ex, tokens, top_k, experts):
    g = _gen(tokens)
    ids = torch.randint(-1, experts + 1, (tokens, top_k), generator=g, dtype=torch.int32)       # repeated, and some that are none
    for r in (ex.plan(ids.cuda(), experts), ex.plan((ids * 0 + experts // 2).cuda(), experts)):
        rows, offsets = ref.order(r.experts.cpu(), experts)
        assert torch.equal(r.rows.cpu(), rows) and torch.equal(r.offsets.cpu(), offsets)


@pytest.mark.parametrize("experts,groups", [(256, 8), (64, 4), (1024, 16), (160, 8)])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_groups_at_the_border_of_what_32_bits_tell_apart(ex, lib, experts, groups, scoring, group_score):
    """Groups of the same logits in another order, but for one bit of one of them: equal, or apart by less than 32 bits show of a score."""
    g = _gen(experts)
    per, tokens = experts // groups, 60
    one = torch.randn((tokens, 1, per), generator=g)
    x = torch.stack([one[:, 0, torch.randperm(per, generator=g)] for _ in range(groups)], 1).contiguous()
    for t in range(tokens):
        for h in torch.randperm(groups, generator=g)[:groups // 2].tolist():
            at = x[t, h].topk(3).indices[t % 3]          # the largest, the second, or one that does not count
            x[t, h, at] = torch.nextafter(x[t, h, at], torch.tensor(INF if t % 2 else -INF))
    x[1, 0] = -INF                                       # groups with one expert and with none
    x[2, 1, 1:] = -INF
    x = x.view(tokens, experts)
    kw = dict(scoring=scoring, groups=groups, top_groups=groups // 2, group_score=group_score)
    bias = torch.full((experts,), 0.125)
    for more in (dict(), dict(bias=bias)):
        r = ex.route(x.cuda(), 6, **kw, **{k: v.cuda() for k, v in more.items()})
        _check_routing(lib, r, x, 6, experts, **kw, **more)


def test_one_bias_for_all_experts(ex, lib):
    g = _gen(8)
    experts, n, k, top_k = 4, 128, 256, 2
    x = torch.randn((30, k), generator=g).half().cuda()
    r = ex.route(torch.randn((30, experts), generator=g).cuda(), top_k)
    w = torch.randint(0, 256, (experts, n, k // 2), generator=g, dtype=torch.uint8).cuda().permute(1, 2, 0)
    w_sf = torch.full((experts, n // 128, k // 64, 32, 4, 4), 0x38, dtype=torch.uint8, device="cuda").permute(3, 4, 1, 5, 2, 0)
    one = torch.randn((1, n), generator=g).half().cuda()
    rows = ex.quantize_routed(x, r)
    y = ex.expert_gemm(rows, r, w, w_sf, bias=one.expand(experts, n))
    assert torch.equal(y, ex.expert_gemm(rows, r, w, w_sf, bias=one.repeat(experts, 1)))
