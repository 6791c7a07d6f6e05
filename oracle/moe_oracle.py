"""Test infrastructure: the operators around the experts' products in plain torch, in 64 bits where values are compared.

Written from the formulas that include/qgemm.h gives; on any device; never on the product path."""
import math

import torch


def route_ref(logits, top_k, bias=None, scoring="softmax", num_groups=1, top_groups=1, group_top=2, renormalize=True, scale=1.0):
    """(weights float64, experts int32, c float64), token by token and pick by pick."""
    T, E = logits.shape
    l = logits.double().cpu()
    s = torch.softmax(l, dim=1) if scoring == "softmax" else torch.sigmoid(l)
    c = s if bias is None else s + bias.double().cpu()
    c = torch.where(l == -math.inf, torch.full_like(c, -math.inf), c)
    order = l if bias is None else c
    n = E // num_groups
    weights, experts = torch.zeros((T, top_k), dtype=torch.float64), torch.full((T, top_k), -1, dtype=torch.int32)

    def before(i, j, v):  # is i picked in front of j
        a, b = float(v[i]), float(v[j])
        if math.isnan(a) or math.isnan(b):
            return math.isnan(a) and (not math.isnan(b) or i < j)
        return a > b or (a == b and i < j)

    def best_of(members, v):
        best = None
        for i in members:
            if best is None or before(i, best, v):
                best = i
        return best

    for t in range(T):
        members = list(range(E))
        if num_groups > top_groups:
            by = order[t] if bias is None and group_top == 1 else c[t]
            worth = []
            for g in range(num_groups):
                left, value = [e for e in range(g * n, g * n + n) if not by[e] == -math.inf], None
                for _ in range(min(group_top, len(left))):
                    e = best_of(left, by)
                    left.remove(e)
                    value = by[e] if value is None else value + by[e]
                worth.append(float("-inf") if value is None else float(value))
            groups = list(range(num_groups))
            for _ in range(num_groups - top_groups):
                worst = groups[0]
                for g in groups[1:]:
                    if before(worst, g, worth):
                        worst = g
                groups.remove(worst)
            members = [e for g in groups for e in range(g * n, g * n + n)]
        members = [e for e in members if not order[t, e] == -math.inf]
        picked = []
        while members and len(picked) < top_k:
            e = best_of(members, order[t])
            members.remove(e)
            picked.append(e)
        if picked:
            w = s[t, picked]
            if renormalize:  # in terms of differences of logits: no sum of zeros
                p = l[t, picked]
                if scoring == "softmax":
                    w = torch.exp(p - p.max())
                elif not float(p.max()) >= -700:
                    w = torch.exp(p - p.max()) if not torch.isnan(p).any() else p
                w = w / w.sum()
            weights[t, :len(picked)] = w * scale
            experts[t, :len(picked)] = torch.tensor(picked, dtype=torch.int32)
    return weights, experts, c


def blocks_ref(experts, num_experts, block_M):
    """(block table without padding entries, rows, sizes), by walking the picks expert by expert."""
    flat = experts.reshape(-1).tolist()
    rows, table, sizes, at = [0] * len(flat), [], [], 0
    mine = [[] for _ in range(num_experts)]
    dropped = []
    for i, e in enumerate(flat):
        (mine[e] if 0 <= e < num_experts else dropped).append(i)
    for e, picks in enumerate(mine):
        sizes.append(len(picks))
        table += [(e, at + i, min(block_M, len(picks) - i)) for i in range(0, len(picks), block_M)]
        for i in picks:
            rows[i] = at
            at += 1
    for i in dropped:
        rows[i] = -2 - at
        at += 1
    return (torch.tensor(table, dtype=torch.int32).reshape(-1, 3), torch.tensor(rows, dtype=torch.int32).reshape(experts.shape),
            torch.tensor(sizes, dtype=torch.int32))


def pow2_ceil(s):
    """The power of two not below a positive fp32 s."""
    m, e = torch.frexp(s.double())
    return torch.where(m == 0.5, s, torch.exp2(e.double()).float())


def swiglu_act_quant_ref(x, round_scale=False):
    """(int8, fp32 scale): everything in 64 bits but the scale, which is rounded to fp32."""
    F = x.shape[-1] // 2
    g, u = x[..., :F].double(), x[..., F:].double()
    a = g / (1 + torch.exp(-g)) * u
    s = (a.abs().amax(dim=-1, keepdim=True).clamp(min=1e-4) / 127.0).float()
    if round_scale:
        s = pow2_ceil(s)
    return torch.round(a / s.double()).clamp(-127, 127).to(torch.int8), s


def combine_ref(y, rows, weights, base=None):
    """(sum, sum of absolute values) in 64 bits."""
    T, k = rows.shape
    out = torch.zeros((T, y.shape[1]), dtype=torch.float64) if base is None else base.double().clone()
    size = out.abs()
    for t in range(T):
        for j in range(k):
            r = int(rows[t, j])
            if 0 <= r < y.shape[0]:
                out[t] += weights[t, j].double() * y[r].double()
                size[t] += (weights[t, j].double() * y[r].double()).abs()
    return out, size
