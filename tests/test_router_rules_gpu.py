"""The router's documented rules where they are easily mistaken: what a bias of zeros changes, and how exact weights are."""
import math

import pytest
import torch

import experts_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nvfp4_gemm_b200 import experts
    return experts


@pytest.mark.parametrize("experts", [16, 64, 256])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_saturated_scores_with_and_without_a_bias_of_zeros(ex, experts, scoring):
    """Scores that are one number in 64 bits: no bias takes the largest logits, a bias of zeros the lowest indices; where
    scores are told apart the two agree."""
    x = torch.arange(experts, dtype=torch.float32) + 40.0               # all sigmoids 1
    if scoring == "softmax":
        x = -1000.0 - 8.0 * torch.arange(experts, dtype=torch.float32).flip(0)       # all but the first expert's score are 0
        x[0] = 5.0
    x = torch.stack([x, torch.randn(experts, generator=torch.Generator().manual_seed(experts))])
    zeros = torch.zeros(experts)
    k = 4
    none = ex.route(x.cuda(), k, scoring=scoring)
    with_zeros = ex.route(x.cuda(), k, scoring=scoring, bias=zeros.cuda())
    high = [experts - 1, experts - 2, experts - 3, experts - 4]
    if scoring == "softmax":
        assert none.experts[0].tolist() == [0] + high[:3] and with_zeros.experts[0].tolist() == [0, 1, 2, 3]
    else:
        assert none.experts[0].tolist() == high and with_zeros.experts[0].tolist() == [0, 1, 2, 3]
    assert none.experts[1].tolist() == with_zeros.experts[1].tolist() == x[1].topk(k).indices.tolist()
    for r, bias in ((none, None), (with_zeros, zeros)):
        assert torch.equal(r.experts.cpu(), ref.route(x, k, scoring=scoring, bias=bias)[0])


@pytest.mark.parametrize("experts,top_k", [(32, 4), (256, 8), (1024, 32)])
@pytest.mark.parametrize("kw", [dict(), dict(renormalize=False), dict(scoring="sigmoid"), dict(scoring="sigmoid", renormalize=False),
                                dict(bias=True), dict(bias=True, renormalize=False), dict(scoring="sigmoid", bias=True)], ids=str)
def test_weights_within_their_documented_error(ex, experts, top_k, kw):
    """A bias that chooses experts far below the largest logit, and many experts a few units below it, where the total's error is largest."""
    g = torch.Generator().manual_seed(experts + top_k)
    x = torch.randn((60, experts), generator=g) * 6
    x[10:30] = torch.randn((20, experts), generator=g) * 0.1 - 5.0
    x[10:30, 3] = 0.0
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = (torch.rand(experts, generator=g) < 0.1).float() * 4 + torch.rand(experts, generator=g)
    r = ex.route(x.cuda(), top_k, **{**kw, **({"bias": kw["bias"].cuda()} if "bias" in kw else {})})
    chosen, weights = ref.route(x, top_k, **kw)
    assert torch.equal(r.experts.cpu(), chosen)
    far = (x.double().gather(1, chosen.long()) - x.double().amax(1, keepdim=True)).abs()
    units = 20.0 if kw.get("scoring") == "sigmoid" else 60.0 + 2.0 * far
    err = (r.weights.cpu().double() - weights).abs()
    normal = weights > 2.0 ** -126
    assert torch.all((err <= units * 2.0 ** -24 * weights) | ~normal), float((err / weights / 2.0 ** -24).max())
    assert math.isfinite(float(err.max()))
