"""Cases of the mixture-of-experts operators and of the matrix product with a residual, with their plain forms.

Five paths, each as a program that serves a model calls it:

* ``route``     router logits -> the experts of each token, their weights, and the order of rows by expert
* ``experts``   tokens and their experts -> the experts' product with bias and (gated) activation, rows in expert order:
                the plan, the 4-bit quantiser into expert order, the grouped product
* ``combine``   rows in expert order -> weighted sum per token, plus the residual stream
* ``residual``  dense 4-bit product with bias, activation and residual
* ``layer``     the whole feed-forward of a layer from logits and hidden states: route, quantise, gate and up product
                re-quantised to 4 bits, down product, combine
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step of a small batch: latency of one call
        {"name": "route_decode_16x64", "op": "route", "tokens": 16, "experts": 64, "top_k": 6, "scoring": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_score": "max", "renormalize": True, "scale": 1.0, "dtype": "bf16"},
        # a prompt's tokens against many experts, with a balancing bias and group-limited choice
        {"name": "route_prefill_8192x256", "op": "route", "tokens": 8192, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_score": "top2", "renormalize": True, "scale": 2.5, "dtype": "fp32"},
        # one sequence being generated: every chosen expert has a token or two, the weights are what is read
        {"name": "experts_decode_4x64_4096x7168", "op": "experts", "tokens": 4, "experts": 64, "top_k": 8, "n": 4096, "k": 7168,
         "activation": "swiglu", "bias": False, "dtype": "bf16"},
        # a batch being generated or a short prompt: ragged counts below a tile, biased experts
        {"name": "experts_batch_333x32_4096x4096", "op": "experts", "tokens": 333, "experts": 32, "top_k": 4, "n": 4096, "k": 4096,
         "activation": "silu", "bias": True, "dtype": "fp16"},
        # the down product of a prompt: short K, wide rows
        {"name": "experts_prefill_4096x32_7168x2048", "op": "experts", "tokens": 4096, "experts": 32, "top_k": 8, "n": 7168, "k": 2048,
         "activation": "none", "bias": False, "dtype": "bf16"},
        # a generated batch's way back into the residual stream
        {"name": "combine_decode_17x7168", "op": "combine", "tokens": 17, "top_k": 8, "n": 7168, "residual": True, "dtype": "bf16"},
        # the same for a prompt
        {"name": "combine_prefill_4096x7168", "op": "combine", "tokens": 4096, "top_k": 8, "n": 7168, "residual": True, "dtype": "fp16"},
        # output projection of a generated batch
        {"name": "residual_decode_17x7168x2048", "op": "residual", "m": 17, "n": 7168, "k": 2048, "l": 1, "activation": "none", "bias": False},
        # output projection of a prompt, with a bias
        {"name": "residual_prefill_4096x7168x7168", "op": "residual", "m": 4096, "n": 7168, "k": 7168, "l": 1, "activation": "none", "bias": True},
        # the feed-forward of one generated token
        {"name": "layer_decode_1x64", "op": "layer", "tokens": 1, "experts": 64, "top_k": 8, "d": 7168, "f": 2048, "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_score": "top2", "renormalize": True, "scale": 2.5, "dtype": "bf16"},
        # ... of a batch of generated tokens
        {"name": "layer_batch_96x32", "op": "layer", "tokens": 96, "experts": 32, "top_k": 4, "d": 4096, "f": 2048, "scoring": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_score": "max", "renormalize": True, "scale": 1.0, "dtype": "bf16"},
        # ... of a long prompt
        {"name": "layer_prefill_8192x32", "op": "layer", "tokens": 8192, "experts": 32, "top_k": 8, "d": 7168, "f": 2048, "scoring": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_score": "max", "renormalize": True, "scale": 1.0, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _router(rng, tokens, experts, top_k):
    groups = rng.choice([1, 1, 4, 8])
    scoring = rng.choice(["softmax", "sigmoid"])
    top_groups = 1 if groups == 1 else rng.choice([g for g in range(1, groups + 1) if g * (experts // groups) >= top_k])
    return {"tokens": tokens, "experts": experts, "top_k": top_k, "scoring": scoring, "bias": rng.random() < 0.5, "groups": groups,
            "top_groups": top_groups, "group_score": rng.choice(["max", "top2"]), "renormalize": rng.random() < 0.7,
            "scale": rng.choice([1.0, 2.5])}


def draw(rng):
    op = rng.choice(["route", "experts", "combine", "residual", "layer"])
    if op == "route":
        experts = rng.choice([8, 16, 40, 64, 128, 256, 384])
        return {"op": op, **_router(rng, _log_int(rng, 1, 8192), experts, rng.randint(1, 8)), "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if op == "experts":
        experts, top_k = rng.choice([8, 16, 32, 64]), rng.randint(1, 8)
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "experts": experts, "top_k": top_k, "n": 128 * rng.randint(2, 48) if rng.random() < 0.5 else 256 * rng.randint(1, 24),
                "k": 256 * rng.randint(1, 24), "activation": rng.choice(["none", "relu", "silu", "swiglu"]), "bias": rng.random() < 0.5,
                "dtype": rng.choice(["fp16", "bf16"])}
    if op == "combine":
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "top_k": rng.randint(1, 8), "n": 128 * rng.randint(1, 56), "residual": rng.random() < 0.7,
                "dtype": rng.choice(["fp16", "bf16"])}
    if op == "residual":
        return {"op": op, "m": _log_int(rng, 1, 4096), "n": 128 * rng.randint(1, 56), "k": 256 * rng.randint(1, 28), "l": rng.choice([1, 1, 2]),
                "activation": rng.choice(["none", "relu", "silu"]), "bias": rng.random() < 0.5}
    experts = rng.choice([8, 16, 32])
    return {"op": op, **_router(rng, _log_int(rng, 1, 4096), experts, rng.randint(1, 8)), "d": 256 * rng.randint(1, 24), "f": 256 * rng.randint(1, 8),
            "dtype": rng.choice(["fp16", "bf16"])}


# ----------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _quantise(v):
    """fp32 [..., K] -> element values (e2m1) and block scales (e4m3 values), both fp32: scale = e4m3(max|v| / 6), element = e2m1(v / scale)."""
    b = v.unflatten(-1, (-1, 16))
    scale = (b.abs().amax(-1, keepdim=True) / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn).float()
    q = torch.where(scale > 0, b / torch.where(scale > 0, scale, 1.0), 0.0)
    a = q.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return ((a / step).round() * step).clamp(max=6.0).copysign(q).flatten(-2), scale.squeeze(-1)


def _quantised(v):
    """fp32 -> the values its 4-bit form stands for."""
    q, scale = _quantise(v)
    return (q.unflatten(-1, (-1, 16)) * scale.unsqueeze(-1)).flatten(-2)


def _pack(q):
    """e2m1 values -> two codes a byte, the lower index in the low nibble."""
    a = q.abs()
    code = torch.where(a <= 2, 2 * a, torch.where(a == 3, 5.0, torch.where(a == 4, 6.0, 7.0))).to(torch.uint8) + 8 * torch.signbit(q).to(torch.uint8)
    code = code.unflatten(-1, (-1, 2))
    return code[..., 0] | (code[..., 1] << 4)


def _operand(g, batch, rows, k, std):
    """A 4-bit matrix per batch entry: codes [rows, K/2, batch], scales [rows, K/16, batch], the same scales in 128 x 4 atoms."""
    packed = torch.empty((batch, rows, k // 2), dtype=torch.uint8, device="cuda")
    sf = torch.empty((batch, rows, k // 16), dtype=torch.float8_e4m3fn, device="cuda")
    for e in range(batch):
        q, scale = _quantise(_randn(g, rows, k) * std)
        packed[e] = _pack(q)
        sf[e] = scale.to(torch.float8_e4m3fn)
    blocks = (rows + 127) // 128
    padded = torch.zeros((batch, blocks * 128, k // 16), dtype=torch.uint8, device="cuda")
    padded[:, :rows] = sf.view(torch.uint8)
    atoms = padded.view(batch, blocks, 4, 32, k // 64, 4).permute(0, 1, 4, 3, 2, 5).contiguous()
    return (packed.permute(1, 2, 0).view(torch.float4_e2m1fn_x2), sf.permute(1, 2, 0),
            atoms.permute(3, 4, 1, 5, 2, 0).view(torch.float8_e4m3fn))


def _logits(g, case):
    # some experts are asked for more often than others, as in a trained router
    x = _randn(g, case["tokens"], case["experts"]) + 0.5 * _randn(g, case["experts"])
    bias = 0.1 * _randn(g, case["experts"]) if case["bias"] else None
    return x, bias


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    op = case["op"]
    if op == "route":
        x, s["router_bias"] = _logits(g, case)
        s["logits"] = x.to(DTYPES[case["dtype"]])
    elif op == "experts":
        t, e, n, k = case["tokens"], case["experts"], case["n"], case["k"]
        liked = _randn(g, t, e) + 0.5 * _randn(g, e)
        s["ids"] = torch.topk(liked, case["top_k"], dim=1).indices.to(torch.int32)
        s["x"] = _randn(g, t, k, dtype=DTYPES[case["dtype"]])
        s["w"] = _operand(g, e, n, k, 1.0)
        s["alpha"] = torch.full((e,), 1.0 / math.sqrt(k), device="cuda")     # the weights' own scale
        s["bias"] = (0.5 * _randn(g, e, n)).half() if case["bias"] else None
    elif op == "combine":
        t, j, n = case["tokens"], case["top_k"], case["n"]
        s["y"] = _randn(g, t * j, n, dtype=torch.float16)
        s["rows"] = torch.randperm(t * j, generator=g, device="cuda").view(t, j).to(torch.int32)
        s["weights"] = torch.softmax(_randn(g, t, j), dim=1)
        s["hidden"] = (2 * _randn(g, t, n)).to(DTYPES[case["dtype"]]) if case["residual"] else None
    elif op == "residual":
        m, n, k, l = case["m"], case["n"], case["k"], case["l"]
        a, b = _operand(g, l, m, k, 1.0), _operand(g, l, n, k, 0.125)
        c = torch.empty((l, m, n), dtype=torch.float16, device="cuda").permute(1, 2, 0)
        s["data"] = (a[0], b[0], a[1], b[1], a[2], b[2], c)
        s["bias"] = _randn(g, n, dtype=torch.float16) if case["bias"] else None
        s["hidden"] = (4 * _randn(g, l, m, n)).half().permute(1, 2, 0)
    else:
        t, e, d, f = case["tokens"], case["experts"], case["d"], case["f"]
        s["logits"], s["router_bias"] = _logits(g, case)
        s["x"] = _randn(g, t, d, dtype=DTYPES[case["dtype"]])
        s["hidden"] = _randn(g, t, d, dtype=DTYPES[case["dtype"]])
        s["up"], s["down"] = _operand(g, e, 2 * f, d, 1.0), _operand(g, e, d, f, 1.0)
        s["up_alpha"] = torch.full((e,), 1.0 / math.sqrt(d), device="cuda")
        s["down_alpha"] = torch.full((e,), 1.0 / math.sqrt(f), device="cuda")
    return s


# ------------------------------------------------------------------------------------------ plain forms
_ELEMENTS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_ELEMENTS = _ELEMENTS + [-v for v in _ELEMENTS]


def _values(packed, sf):
    """Codes [B, rows, K/2] and scales [B, rows, K/16] -> fp32 [B, rows, K]."""
    pairs = torch.tensor([[_ELEMENTS[b & 15], _ELEMENTS[b >> 4]] for b in range(256)], device=packed.device)
    v = pairs.index_select(0, packed.reshape(-1).int()).view(*packed.shape[:2], -1, 16)
    return (v * sf.float().unsqueeze(-1)).flatten(-2)


def _codes(t):
    return t.view(torch.uint8).permute(2, 0, 1)


def _order(ids, experts):
    """Pairs in expert order (stable): the order, each pair's row, the experts' first rows."""
    flat = ids.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    rows = torch.empty_like(order)
    rows[order] = torch.arange(flat.numel(), device=flat.device)
    counts = (flat.unsqueeze(1) == torch.arange(experts, device=flat.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return order, rows.view(ids.shape).to(torch.int32), offsets.to(torch.int32)


def _choose(case, logits, bias):
    """The experts and their weights.  In 64 bits: two scores may be as near to each other as their 32-bit rounding."""
    x = logits.double()
    scores = torch.softmax(x, 1) if case["scoring"] == "softmax" else torch.sigmoid(x)
    choice = scores + bias.double() if bias is not None else scores
    if case["groups"] > 1:
        grouped = choice.unflatten(1, (case["groups"], -1))
        top = grouped.topk(min(2, grouped.shape[2]) if case["group_score"] == "top2" else 1, dim=2).values.sum(2)
        best = torch.sort(top, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros_like(top, dtype=torch.bool).scatter(1, best, True)
        choice = torch.where(keep.unsqueeze(2), grouped, -math.inf).flatten(1)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
    w = scores.gather(1, ids)
    if case["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return ids.to(torch.int32), (w * case["scale"]).float()


def _expert_product(x, order, ids, top_k, w, alpha, bias, by_row=False):
    """Rows in expert order: alpha_e * x W_e^T + bias_e, in 32 bits.  x: per token, or per row already."""
    packed, sf = _codes(w[0]), w[1].permute(2, 0, 1)
    expert = ids.reshape(-1).long()[order]
    rows = x if by_row else x[order // top_k]
    experts = packed.shape[0]
    if expert.numel() <= experts:
        z = torch.bmm(_values(packed[expert], sf.view(torch.uint8)[expert].view(torch.float8_e4m3fn)), rows.unsqueeze(2)).squeeze(2)
    else:
        counts = torch.bincount(expert, minlength=experts)
        place = torch.arange(expert.numel(), device=x.device) - (counts.cumsum(0) - counts)[expert]
        padded = rows.new_zeros(experts, int(counts.max()), rows.shape[1])
        padded[expert, place] = rows
        z = torch.bmm(padded, _values(packed, sf).transpose(1, 2))[expert, place]
    z = z * alpha[expert].unsqueeze(1)
    return z + bias.float()[expert] if bias is not None else z


def _silu(z):
    return z * torch.sigmoid(z)


def _activate(z, activation):
    if activation == "swiglu":      # gate and up columns alternate in groups of eight
        pairs = z.unflatten(-1, (-1, 2, 8))
        return (_silu(pairs[..., 0, :]) * pairs[..., 1, :]).flatten(-2)
    return torch.relu(z) if activation == "relu" else _silu(z) if activation == "silu" else z


def _combined(y, rows, weights, hidden, dtype):
    total = (y.float()[rows.long()] * weights.unsqueeze(2)).sum(1)
    return (total + hidden.float() if hidden is not None else total).to(dtype)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "route":
        ids, weights = _choose(case, s["logits"], s["router_bias"])
        _, rows, offsets = _order(ids, case["experts"])
        return {"experts": ids, "weights": weights, "rows": rows, "offsets": offsets}
    if op == "experts":
        order, _, _ = _order(s["ids"], case["experts"])
        z = _expert_product(_quantised(s["x"].float()), order, s["ids"], case["top_k"], s["w"], s["alpha"], s["bias"])
        return _activate(z, case["activation"]).half()
    if op == "combine":
        return _combined(s["y"], s["rows"], s["weights"], s["hidden"], DTYPES[case["dtype"]])
    if op == "residual":
        a, b, sfa, sfb = s["data"][:4]
        z = torch.bmm(_values(_codes(a), sfa.permute(2, 0, 1)), _values(_codes(b), sfb.permute(2, 0, 1)).transpose(1, 2))
        z = z + s["bias"].float() if s["bias"] is not None else z
        return (_activate(z, case["activation"]).permute(1, 2, 0) + s["hidden"].float()).half()
    ids, weights = _choose(case, s["logits"], s["router_bias"])
    order, rows, _ = _order(ids, case["experts"])
    z = _expert_product(_quantised(s["x"].float()), order, ids, case["top_k"], s["up"], s["up_alpha"], None)
    h = _quantised(_activate(z, "swiglu").half().float())
    y = _expert_product(h, order, ids, case["top_k"], s["down"], s["down_alpha"], None, by_row=True).half()
    return _combined(y, rows, weights, s["hidden"], DTYPES[case["dtype"]])


def _router_arguments(s):
    c = s["case"]
    return dict(scoring=c["scoring"], bias=s["router_bias"], groups=c["groups"], top_groups=c["top_groups"], group_score=c["group_score"],
                renormalize=c["renormalize"], scale=c["scale"])


def _own(s):
    from nvfp4_gemm_b200 import experts, submission
    case = s["case"]
    op = case["op"]
    if op == "route":
        r = experts.route(s["logits"], case["top_k"], **_router_arguments(s))
        return {"experts": r.experts, "weights": r.weights, "rows": r.rows, "offsets": r.offsets}
    if op == "experts":
        r = experts.plan(s["ids"], case["experts"])
        return experts.expert_gemm(experts.quantize_routed(s["x"], r), r, s["w"][0], s["w"][2], alpha=s["alpha"], bias=s["bias"],
                                   activation=case["activation"])
    if op == "combine":
        return experts.combine(s["y"], s["rows"], s["weights"], residual=s["hidden"], dtype=DTYPES[case["dtype"]])
    if op == "residual":
        return submission.gemm_epilogue(s["data"], bias=s["bias"], activation=case["activation"], residual=s["hidden"])
    return experts.expert_layer(s["x"], s["logits"], (s["up"][0], s["up"][2]), (s["down"][0], s["down"][2]), case["top_k"],
                                up_alpha=s["up_alpha"], down_alpha=s["down_alpha"], residual=s["hidden"], **_router_arguments(s))


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------- work
_BYTES_4BIT = 0.5625      # half a byte an element, a byte of scale for 16


def _touched(tokens, top_k, experts):
    """Experts that some token chooses, on average when all are as likely."""
    return experts * (1.0 - (1.0 - top_k / experts) ** tokens)


def work(case):
    op = case["op"]
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": t * e * DTYPES[case["dtype"]].itemsize + (4 * e if case["bias"] else 0) + 12 * t * k + 4 * (e + 1), "flops": 8 * t * e}
    if op == "experts":
        t, j, n, k = case["tokens"], case["top_k"], case["n"], case["k"]
        used = _touched(t, j, case["experts"])
        out = n // 2 if case["activation"] == "swiglu" else n
        return {"bytes": 2 * t * k + 4 * t * j + used * n * k * _BYTES_4BIT + (used * 2 * n if case["bias"] else 0) + 2 * t * j * out, "flops": 2 * t * j * n * k}
    if op == "combine":
        t, j, n = case["tokens"], case["top_k"], case["n"]
        return {"bytes": 2 * t * j * n + 8 * t * j + 2 * t * n * (2 if case["residual"] else 1), "flops": 2 * t * j * n}
    if op == "residual":
        m, n, k, l = case["m"], case["n"], case["k"], case["l"]
        return {"bytes": l * ((m + n) * k * _BYTES_4BIT + 4 * m * n) + (2 * n if case["bias"] else 0), "flops": 2 * l * m * n * k}
    t, e, j, d, f = case["tokens"], case["experts"], case["top_k"], case["d"], case["f"]
    return {"bytes": 4 * t * e + 2 * t * d * 3 + _touched(t, j, e) * 3 * f * d * _BYTES_4BIT, "flops": 6 * t * j * d * f}


# ------------------------------------------------------------------------------------------------ exact
def _exact_quantised(v):
    """float64 values of the 4-bit form: thresholds between neighbouring values instead of a rounded quotient."""
    b = v.reshape(*v.shape[:-1], v.shape[-1] // 16, 16)
    scale = torch.clamp(b.abs().max(-1, keepdim=True).values / 6, max=448).to(torch.float8_e4m3fn).double()
    ends = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=v.device)
    a = b.abs()
    index = torch.zeros(b.shape, dtype=torch.uint8, device=v.device)
    for i in range(7):      # a tie goes to the value with the even code
        index += (a >= ends[i] * scale) if i % 2 else (a > ends[i] * scale)
    value = torch.tensor(_ELEMENTS[:8], dtype=torch.float64, device=v.device).index_select(0, index.reshape(-1).int()).view(b.shape)
    return (torch.where(scale > 0, value * scale, 0.0) * torch.where(b < 0, -1.0, 1.0)).reshape(v.shape)


def _exact_values(t, sf, e):
    """Entry e of a 4-bit operand in float64 [rows, K]."""
    c = t.view(torch.uint8)[:, :, e].int()
    codes = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    mantissa, exponent = (codes & 1).double(), ((codes >> 1) & 3).double()
    v = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * torch.exp2(exponent - 1))
    return torch.where(codes >= 8, -v, v) * sf[:, :, e].double().repeat_interleave(16, dim=1)


def _exact_choose(case, logits, bias):
    x = logits.double()
    if case["scoring"] == "softmax":
        p = torch.exp(x - x.max(1, keepdim=True).values)
        scores = p / p.sum(1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-x))
    choice = scores.clone() if bias is None else scores + bias.double()
    t, e = choice.shape
    per = e // case["groups"]
    if case["groups"] > 1:
        ranked = choice.view(t, case["groups"], per).sort(2, descending=True).values
        value = ranked[:, :, 0] + (ranked[:, :, 1] if case["group_score"] == "top2" and per > 1 else 0)
        rank = (value.unsqueeze(1) > value.unsqueeze(2)).sum(2)
        choice = torch.where((rank < case["top_groups"]).repeat_interleave(per, dim=1), choice, -math.inf)
    picked = []
    for _ in range(case["top_k"]):
        picked.append(choice.argmax(1))
        choice = choice.scatter(1, picked[-1].unsqueeze(1), -math.inf)
    ids = torch.stack(picked, 1)
    w = torch.gather(scores, 1, ids)
    if case["renormalize"]:
        w = w / w.sum(1, keepdim=True)
    return ids, w * case["scale"]


def _exact_expert(x, e, w, alpha, bias):
    z = alpha[e].double() * (x @ _exact_values(w[0], w[1], e).t())
    return z if bias is None else z + bias[e].double()


def _exact_activate(z, activation):
    if activation == "relu":
        return z.clamp(min=0)
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    if activation == "swiglu":
        rows, n = z.shape
        p = z.reshape(rows, n // 16, 16)
        gate, up = p[:, :, :8], p[:, :, 8:]
        return (gate / (1 + torch.exp(-gate)) * up).reshape(rows, n // 2)
    return z


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        ids, w = _exact_choose(case, s["logits"], s["router_bias"])
        return {"experts": ids.to(torch.int32), "weights": w, "rows": None, "offsets": None}
    if op == "combine":
        total = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device="cuda")
        for j in range(case["top_k"]):
            total += s["weights"][:, j:j + 1].double() * s["y"][s["rows"][:, j].long()].double()
        return total if s["hidden"] is None else total + s["hidden"].double()
    if op == "residual":
        a, b, sfa, sfb = s["data"][:4]
        out = torch.empty(case["m"], case["n"], case["l"], dtype=torch.float64, device="cuda")
        for i in range(case["l"]):
            z = _exact_values(a, sfa, i) @ _exact_values(b, sfb, i).t()
            z = z if s["bias"] is None else z + s["bias"].double()
            out[:, :, i] = _exact_activate(z, case["activation"]) + s["hidden"][:, :, i].double()
        return out
    if op == "experts":
        x = _exact_quantised(s["x"].double())
        parts = []
        for e in range(case["experts"]):
            tokens = (s["ids"] == e).any(1).nonzero().squeeze(1)      # a token takes an expert once
            parts.append(_exact_activate(_exact_expert(x[tokens], e, s["w"], s["alpha"], s["bias"]), case["activation"]))
        return torch.cat(parts)
    ids, w = _exact_choose(case, s["logits"], s["router_bias"])
    x = _exact_quantised(s["x"].double())
    out = s["hidden"].double()
    for e in range(case["experts"]):
        tokens, slot = (ids == e).nonzero(as_tuple=True)
        h = _exact_activate(_exact_expert(x[tokens], e, s["up"], s["up_alpha"], None), "swiglu")
        y = _exact_expert(_exact_quantised(h.half().double()), e, s["down"], s["down_alpha"], None)
        out.index_add_(0, tokens, w[tokens, slot].unsqueeze(1) * y.half().double())
    return out
