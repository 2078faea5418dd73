"""The mixture-of-experts operators in 64 bits, written for reading (what the kernels are compared with)."""
import math

import torch

E2M1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def values(packed, sf):
    """codes [..., K/2], scales [..., K/16] (bytes) -> float64 [..., K]"""
    c = packed.view(torch.uint8).long()
    v = E2M1.to(c.device)[torch.stack([c & 15, c >> 4], -1)].flatten(-2)
    return v * sf.view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)


def route(logits, top_k, scoring="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0):
    """One token at a time, on the CPU.  -> experts [T, k] (-1: none), weights float64"""
    x_all = logits.double().cpu()
    experts, weights = [], []
    for x in x_all.tolist():
        x = [-math.inf if math.isnan(v) else min(v, 3.4028234663852886e38) for v in x]
        free = [e for e, v in enumerate(x) if v != -math.inf]
        if scoring == "softmax":
            top = max(x)
            total = sum(math.exp(x[e] - top) for e in free)
            s = [math.exp(v - top) / total if v != -math.inf else 0.0 for v in x]
        else:
            s = [1 / (1 + math.exp(-v)) if v > -700 else 0.0 for v in x]
        # choice: the score with its bias; without one the order of the logits, which both scores keep
        judged = s if bias is not None or (groups > 1 and group_score == "top2") else x
        b = bias.double().tolist() if bias is not None else [0.0] * len(x)
        c = {e: judged[e] + b[e] for e in free if not math.isnan(b[e]) and b[e] != -math.inf}
        if groups > 1:
            per = len(x) // groups
            judge = {}
            for g in range(groups):
                best = sorted((c[e] for e in range(g * per, (g + 1) * per) if e in c), reverse=True)
                if best:
                    judge[g] = best[0] + (best[1] if group_score == "top2" and len(best) > 1 else 0.0)
            kept = sorted(judge, key=lambda g: (-judge[g], g))[:top_groups]
            c = {e: v for e, v in c.items() if e // per in kept}
        ids = sorted(c, key=lambda e: (-c[e], e))[:top_k]
        w = [s[e] for e in ids]
        if renormalize:
            total = sum(w)
            w = [v / total if total > 0 else 0.0 for v in w]
        experts.append(ids + [-1] * (top_k - len(ids)))
        weights.append([v * scale for v in w] + [0.0] * (top_k - len(ids)))
    return torch.tensor(experts, dtype=torch.int32).view(-1, top_k), torch.tensor(weights, dtype=torch.float64).view(-1, top_k)


def order(experts, num_experts):
    """-> rows [T, k] (-1: none), offsets [E + 1], on the CPU"""
    flat = experts.cpu().reshape(-1).tolist()
    lists = [[] for _ in range(num_experts)]
    for i, e in enumerate(flat):
        if 0 <= e < num_experts:
            lists[e].append(i)
    rows, offsets, at = [-1] * len(flat), [0], 0
    for members in lists:
        for i in members:
            rows[i] = at
            at += 1
        offsets.append(at)
    return torch.tensor(rows, dtype=torch.int32).view(experts.shape), torch.tensor(offsets, dtype=torch.int32)


def sf_rows(offsets, tile_tokens):
    """Row of each expert-order row in the scales' atoms: every token tile starts a block of 128."""
    block = (tile_tokens + 127) // 128 * 128
    out, tile = [], 0
    o = offsets.tolist()
    for e in range(len(o) - 1):
        for i in range(o[e + 1] - o[e]):
            out.append((tile + i // tile_tokens) * block + i % tile_tokens)
        tile += (o[e + 1] - o[e] + tile_tokens - 1) // tile_tokens
    return torch.tensor(out, dtype=torch.long)


def scales_of(sf, where, k):
    """The scale bytes [rows, K/16] of rows at `where` of the atoms [blocks][K/64][32][4][4]."""
    atoms = sf.view(torch.uint8).view(-1, k // 64, 32, 4, 4)
    w = where.to(sf.device)
    return atoms[w // 128, :, w % 32, (w % 128) // 32].reshape(len(w), k // 16)


def activate(z, activation):
    if activation == "swiglu":
        p = z.unflatten(-1, (-1, 2, 8))
        g, u = p[..., 0, :], p[..., 1, :]
        return (g / (1 + torch.exp(-g)) * u).flatten(-2)
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    return z.clamp(min=0) if activation == "relu" else z


def expert_product(a, offsets, w, alpha, bias):
    """a: float64 rows in expert order [R, K]; w: float64 [E, N, K].  -> z [R, N] and the sum of the absolute products."""
    z, size = [], []
    for e in range(w.shape[0]):
        rows = a[offsets[e]:offsets[e + 1]]
        f = float(alpha[e]) if alpha is not None else 1.0
        b = bias[e].double() if bias is not None else 0.0
        z.append(f * (rows @ w[e].t()) + b)
        size.append(abs(f) * (rows.abs() @ w[e].abs().t()) + (b.abs() if bias is not None else 0.0))
    return torch.cat(z), torch.cat(size)
