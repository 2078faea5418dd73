"""The experts' operators where elements and bytes are counted beyond 32 bits: what stands there equals what a small call makes of the same rows."""
import pytest
import torch

from test_experts_gpu import _weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    from nvfp4_gemm_b200 import experts
    yield experts
    torch.cuda.empty_cache()


def test_rows_beyond_2_to_the_31(ex):
    """330 000 tokens, two choices each of four experts: 660 000 rows of 7168 columns are 4.7e9 values; the last tokens are the first again."""
    tokens, top_k, experts, k, n = 330_000, 2, 4, 256, 7168
    few = 500
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((tokens, k), generator=g, device="cuda").bfloat16()
    logits = torch.randn((tokens, experts), generator=g, device="cuda")
    x[-few:], logits[-few:] = x[:few], logits[:few]
    w, w_sf, _ = _weights(experts, n, k, 2)
    alpha = torch.full((experts,), 2.0 ** -6, device="cuda")
    r, small = ex.route(logits, top_k), ex.route(logits[:few], top_k)
    assert torch.equal(r.experts[-few:], small.experts) and int(r.offsets[-1]) == tokens * top_k
    assert torch.equal(r.rows.flatten().sort().values, torch.arange(tokens * top_k, device="cuda", dtype=torch.int32))
    rows, some = ex.quantize_routed(x, r), ex.quantize_routed(x[:few], small)
    y, z = ex.expert_gemm(rows, r, w, w_sf, alpha=alpha), ex.expert_gemm(some, small, w, w_sf, alpha=alpha)
    assert y.numel() > 2 ** 32
    for part in (slice(0, few), slice(tokens - few, tokens)):
        at = r.rows[part].long().flatten()
        assert int(at.max()) * n > 2 ** 31
        assert torch.equal(rows.packed.view(torch.uint8)[at], some.packed.view(torch.uint8)[small.rows.long().flatten()])
        assert torch.equal(y[at], z[small.rows.long().flatten()])
    q, p = ex.expert_gemm(rows, r, w, w_sf, alpha=alpha, nvfp4_out=True), ex.expert_gemm(some, small, w, w_sf, alpha=alpha, nvfp4_out=True)
    assert q.packed.numel() > 2 ** 31
    for part in (slice(0, few), slice(tokens - few, tokens)):
        assert torch.equal(q.packed.view(torch.uint8)[r.rows[part].long().flatten()], p.packed.view(torch.uint8)[small.rows.long().flatten()])
    # the re-quantised rows through a following product: their scales are found again, wherever they stand
    v, v_sf, _ = _weights(experts, 128, n, 3)
    last, first = ex.expert_gemm(q, r, v, v_sf, alpha=alpha), ex.expert_gemm(p, small, v, v_sf, alpha=alpha)
    for part in (slice(0, few), slice(tokens - few, tokens)):
        assert torch.equal(last[r.rows[part].long().flatten()], first[small.rows.long().flatten()])
    del q, p, last, first
    out = ex.combine(y, r.rows, r.weights, dtype=torch.bfloat16)
    assert out.numel() > 2 ** 31
    exp = ex.combine(z, small.rows, small.weights, dtype=torch.bfloat16)
    assert torch.equal(out[:few], exp) and torch.equal(out[-few:], exp)


def test_logits_beyond_2_to_the_31(ex):
    tokens, experts, top_k, few = 2_200_000, 1024, 4, 3000
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn((tokens, experts), generator=g, device="cuda", dtype=torch.bfloat16)
    logits[-few:] = logits[:few]
    assert logits.numel() > 2 ** 31
    for kw in (dict(), dict(scoring="sigmoid", bias=torch.zeros(experts, device="cuda"))):
        r, small = ex.route(logits, top_k, **kw), ex.route(logits[:few], top_k, **kw)
        for part in (slice(0, few), slice(tokens - few, tokens)):
            assert torch.equal(r.experts[part], small.experts) and torch.equal(r.weights[part], small.weights)
        count = torch.bincount(r.experts.flatten(), minlength=experts)
        assert torch.equal(r.offsets.long(), torch.cat([count.new_zeros(1), count.cumsum(0)]))
        assert torch.equal(r.rows.flatten().sort().values, torch.arange(tokens * top_k, device="cuda", dtype=torch.int32))
        # by expert, within an expert by token and choice
        stable = torch.sort(r.experts.flatten(), stable=True).indices
        assert torch.equal(r.rows.flatten()[stable], torch.arange(tokens * top_k, device="cuda", dtype=torch.int32))
