"""What the mixture-of-experts operators refuse, before any GPU is touched, and their host-side sizes."""
import ctypes

import pytest
import torch

from nvfp4_gemm_b200 import _lib, experts

A = 0x10000          # an aligned address that nothing reads: every call below is refused on the host


def _routing(**over):
    r = _lib.RoutingStruct(8, 2, 16, A, A, A, A)
    for k, v in over.items():
        setattr(r, k, v)
    return r


def _router(**over):
    o = _lib.Router(A, _lib.LOGITS_FP32, 16, None, _lib.SCORE_SOFTMAX, 1, 1, 1, 1, 1.0, A)
    for k, v in over.items():
        setattr(o, k, v)
    return o


def _problem(**over):
    p = _lib.ExpertProblem(A, A, A, A, None, None, 256, 512, 256, 256, 256 * 256, 2 * 8 * 512, 0, 0, 0, 1.0, A, 256, None)
    for k, v in over.items():
        setattr(p, k, v)
    return p


def _refused(lib, rc, text):
    assert rc == _lib.NVFP4_ERR_INVALID_ARGUMENT
    assert text in lib.nvfp4_last_error().decode(), lib.nvfp4_last_error()


@pytest.mark.parametrize("router,routing,text", [
    (dict(logits=None), dict(), "must not be NULL"),
    (dict(weights=None), dict(), "must not be NULL"),
    (dict(logits_type=3), dict(), "logits_type"),
    (dict(logits=A + 2), dict(), "aligned"),
    (dict(scoring=2), dict(), "scoring"),
    (dict(groups=3), dict(), "groups must divide"),
    (dict(groups=4, top_groups=5), dict(), "top_groups"),
    (dict(groups=8, top_groups=0), dict(), "top_groups"),
    (dict(groups=64, top_groups=1), dict(experts=64), "groups"),
    (dict(group_top=3), dict(), "group_top"),
    (dict(groups=8, top_groups=1), dict(top_k=3), "top_k = 3 of the 2 experts"),
    (dict(), dict(top_k=17), "top_k = 17 of 16"),
    (dict(), dict(top_k=0), "positive"),
    (dict(), dict(tokens=-1), "negative"),
    (dict(), dict(experts=2048), "at most 1024"),
    (dict(), dict(top_k=33, experts=64), "top_k 32"),
    (dict(), dict(tokens=2 ** 30, top_k=4), "too large"),
    (dict(), dict(plan=None), "plan"),
    (dict(), dict(plan=A + 8), "plan"),
    (dict(), dict(expert=None), "must not be NULL"),
])
def test_router_refusals(lib, router, routing, text):
    _refused(lib, lib.nvfp4_route(_router(**router), _routing(**routing), None), text)


def test_null_structs(lib):
    _refused(lib, lib.nvfp4_route(None, _routing(), None), "router is NULL")
    _refused(lib, lib.nvfp4_route(_router(), None, None), "routing is NULL")
    _refused(lib, lib.nvfp4_expert_gemm(None, _routing(), None), "problem is NULL")
    _refused(lib, lib.nvfp4_plan_experts(_routing(row=None), None), "must not be NULL")


@pytest.mark.parametrize("over,text", [
    (dict(n=200), "multiple of 128"), (dict(n=0), "multiple of 128"), (dict(k=384), "multiple of 256"), (dict(a=None), "must not be NULL"),
    (dict(w=A + 8), "16-byte aligned"), (dict(bias=A + 1), "aligned"), (dict(alpha=A + 2), "aligned"), (dict(activation=4), "activation"),
    (dict(output=2), "output"), (dict(output=1), "out_sf"), (dict(a_row_stride=200), "row strides"), (dict(w_row_stride=128), "row strides"),
    (dict(w_expert_stride=24), "expert strides"), (dict(sfw_perm_expert_stride=-16), "expert strides"), (dict(out_row_stride=128), "out_row_stride"),
    (dict(out_row_stride=260), "out_row_stride"),
])
def test_grouped_product_refusals(lib, over, text):
    _refused(lib, lib.nvfp4_expert_gemm(_problem(**over), _routing(), None), text)


@pytest.mark.parametrize("over", [dict(w_expert_stride=0), dict(sfw_perm_expert_stride=0), dict(w_expert_stride=16), dict(bias_expert_stride=-8)])
def test_experts_that_share_weights_are_refused(lib, over):
    _refused(lib, lib.nvfp4_expert_gemm(_problem(bias=A, **over), _routing(), None), "expert strides")


@pytest.mark.parametrize("args,text", [
    (dict(k=96), "multiple of 64"), (dict(x=None), "must not be NULL"), (dict(x=A + 8), "16-byte aligned"), (dict(stride=252), "row stride"),
    (dict(packed=A + 4), "packed"), (dict(packed_stride=100), "packed"), (dict(sf=A + 8), "16-byte aligned"),
])
def test_routed_quantiser_refusals(lib, args, text):
    a = {**dict(x=A, stride=256, k=256, packed=A, packed_stride=128, sf=A), **args}
    _refused(lib, lib.nvfp4_quantize_routed(a["x"], 0, a["stride"], a["k"], _routing(), a["packed"], a["packed_stride"], a["sf"], None), text)


@pytest.mark.parametrize("args,text", [
    (dict(n=12), "multiple of 8"), (dict(top_k=33), "top_k"), (dict(tokens=-1), "negative"), (dict(y=None), "must not be NULL"),
    (dict(out=A + 8), "16-byte aligned"), (dict(out_stride=8), "at least n"), (dict(residual_stride=12), "row strides"),
])
def test_combination_refusals(lib, args, text):
    a = {**dict(y=A, y_rows=4, row=A, weights=A, tokens=2, top_k=2, n=16, residual=A, residual_stride=16, out=A, out_stride=16), **args}
    _refused(lib, lib.nvfp4_combine_experts(a["y"], 16, a["y_rows"], a["row"], a["weights"], a["tokens"], a["top_k"], a["n"], a["residual"],
                                            a["residual_stride"], a["out"], a["out_stride"], 0, None), text)


@pytest.mark.parametrize("tokens,top_k,num_experts", [(0, 1, 1), (1, 1, 1), (1, 8, 256), (37, 3, 8), (4096, 8, 32), (8192, 8, 256), (100000, 1, 1024)])
def test_plan_sizes_hold_every_distribution(lib, tokens, top_k, num_experts):
    """The scales' memory covers the tiles of the distribution with most of them: one row more than full tiles in as many experts as can be."""
    tile, plan_bytes, sf_rows = ctypes.c_int32(), ctypes.c_int64(), ctypes.c_int64()
    assert lib.nvfp4_routing_plan(tokens, top_k, num_experts, ctypes.byref(tile), ctypes.byref(plan_bytes), ctypes.byref(sf_rows)) == 0
    pairs, t = tokens * top_k, tile.value
    used = min(pairs, num_experts)
    most = used + (pairs - used) // t                     # a row in each, then full tiles more
    block = (t + 127) // 128 * 128
    assert sf_rows.value >= most * block
    assert plan_bytes.value >= 4 * (4 + 4 * most + pairs)
    assert lib.nvfp4_routing_plan(tokens, top_k, num_experts, None, None, None) == 0


def test_python_refusals(lib):
    x, ids = torch.zeros((4, 256), dtype=torch.bfloat16), torch.zeros((4, 2), dtype=torch.int32)
    r = experts.Routing(ids, None, ids, ids, ids, 8)
    for call in (lambda: experts.route(torch.zeros((4, 8)), 2), lambda: experts.plan(ids, 8), lambda: experts.quantize_routed(x, r),
                 lambda: experts.expert_gemm((x, x), r, x, x), lambda: experts.combine(x.half(), ids, x)):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError, match="scoring must be one of 'softmax', 'sigmoid'"):
        experts.route(torch.zeros((4, 8)), 2, scoring="relu")
    with pytest.raises(ValueError, match="activation"):
        experts.expert_gemm((x, x), r, x, x, activation="gelu")
    with pytest.raises(ValueError, match="fp16 or bf16"):
        experts.combine(x, ids, x, dtype=torch.float32)
    with pytest.raises(TypeError, match="logits must be a tensor"):
        experts.route([1.0], 1)


def test_interleaving_gate_and_up():
    gate, up = torch.arange(64).view(64, 1), torch.arange(100, 164).view(64, 1)
    rows = experts.interleave_gate_up(gate, up).view(-1).tolist()
    assert rows[:24] == list(range(8)) + list(range(100, 108)) + list(range(8, 16))
    with pytest.raises(ValueError, match="multiple of 64"):
        experts.interleave_gate_up(gate[:32], up[:32])
