"""Performance cases of the operators around the experts' products of a mixture layer.

Between a router's logits and the grouped int8 products, and behind them, a layer picks experts for each token, sorts the
picks by expert into the row blocks that the products take, quantises each token's row into its places, joins the two
products by a gated activation that is quantised again, and adds the outputs up per token.  Five kinds, one for each:

``route``     logits [tokens, experts] -> the weights and the indices of the experts picked
``blocks``    the picked experts -> the table of row blocks, each pick's place in the stacked rows, rows per expert
``dispatch``  bf16 / f16 rows -> int8 rows and scales, each at all the places of its token
``gate``      gate and up projections side by side -> their SiLU-gated product as int8 rows and scales
``combine``   expert outputs in the stacked order -> the weighted sum per token, on top of a base where there is one

The int8 values are the operands of an exact integer product, so they come back as the whole numbers that they are, and
the scales beside them.  Where a value lies next to a border - a pick between two nearly equal scores, a quotient half-way between two
integers - the definition's real numbers decide, so the plain forms of ``route`` and ``gate`` are computed in 64 bits.
"""
import math

import torch

own = False

_DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}


def _route(tokens, experts, k, scoring, dtype, bias=False, groups=1, top_groups=1, group_top=2, renormalize=True, scale=1.0):
    return {"kind": "route", "tokens": tokens, "experts": experts, "k": k, "scoring": scoring, "dtype": dtype, "bias": bias,
            "groups": groups, "top_groups": top_groups, "group_top": group_top, "renormalize": renormalize, "scale": scale}


def _blocks(tokens, experts, k, block=128, dropped=0.0):
    return {"kind": "blocks", "tokens": tokens, "experts": experts, "k": k, "block": block, "dropped": dropped}


def _dispatch(tokens, width, experts, k, dtype="bfloat16", round_scale=False, dropped=0.0):
    return {"kind": "dispatch", "tokens": tokens, "width": width, "experts": experts, "k": k, "dtype": dtype, "round_scale": round_scale,
            "dropped": dropped}


def _gate(rows, width, dtype="bfloat16", round_scale=False):
    return {"kind": "gate", "rows": rows, "width": width, "dtype": dtype, "round_scale": round_scale}


def _combine(tokens, width, experts, k, dtype="bfloat16", base=False, dropped=0.0):
    return {"kind": "combine", "tokens": tokens, "width": width, "experts": experts, "k": k, "dtype": dtype, "base": base, "dropped": dropped}


def listed():
    return [
        # one decode step of 16 sequences: sigmoid scores, a bias for balance, the best four of eight groups; latency
        dict(_route(16, 256, 8, "sigmoid", "float32", True, 8, 4, scale=2.5), name="route_decode"),
        # the same router over a long prefill chunk
        dict(_route(16384, 256, 8, "sigmoid", "bfloat16", True, 8, 4, scale=2.5), name="route_prefill"),
        # a softmax router of few experts without groups, ragged number of tokens
        dict(_route(4099, 60, 4, "softmax", "float32"), name="route_softmax"),
        # tables of a decode step of 16 sequences
        dict(_blocks(16, 256, 8), name="blocks_decode"),
        # ... of a long prefill chunk
        dict(_blocks(16384, 256, 8), name="blocks_prefill"),
        # one decode step: the tokens' rows quantised into the experts' order
        dict(_dispatch(16, 7168, 256, 8), name="dispatch_decode"),
        # a prefill chunk of ragged length, two experts each
        dict(_dispatch(4001, 4096, 16, 2, "float16"), name="dispatch_two"),
        # a prefill chunk, eight experts each
        dict(_dispatch(4096, 7168, 256, 8), name="dispatch_prefill"),
        # between the two products of a decode step: 128 rows
        dict(_gate(128, 2048), name="gate_decode"),
        # ... of a prefill chunk
        dict(_gate(32768, 2048), name="gate_prefill"),
        # outputs of a decode step summed on top of the shared expert's
        dict(_combine(16, 7168, 256, 8, base=True), name="combine_decode"),
        # ... of a prefill chunk
        dict(_combine(4096, 7168, 256, 8), name="combine_prefill"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], uniform in its logarithm."""
    x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(x / step)) * step))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0), _cost(c))
    kind = rng.choice(["route", "route", "blocks", "dispatch", "gate", "combine"])
    while True:
        half = rng.choice(["float16", "bfloat16"])
        k = rng.randint(1, 10)
        if kind == "route":
            groups = rng.choice([1, 1, 2, 4, 8, 12])
            experts = groups * rng.randint(-(-max(k, 4) // groups), max(16, 384 // groups))
            top_groups = groups if groups == 1 else rng.randint(-(-groups // 2), groups)
            if experts // groups * top_groups < k:
                continue
            bias = rng.random() < 0.5
            case = _route(_log(rng, 1, 20000), experts, k, rng.choice(["softmax", "sigmoid"]), rng.choice(["float32", "bfloat16", "float16"]),
                          bias, groups, top_groups, rng.choice([1, 2]), rng.random() < 0.7, rng.choice([1.0, 2.5]))
        elif kind == "blocks":
            case = _blocks(_log(rng, 1, 30000), rng.randint(max(k, 4), 400), k, rng.choice([128, 128, 64]), rng.choice([0.0, 0.0, 0.05]))
        elif kind == "dispatch":
            case = _dispatch(_log(rng, 1, 8192), _log(rng, 512, 8192, 8), rng.randint(max(k, 4), 256), k, half, rng.random() < 0.3,
                             rng.choice([0.0, 0.0, 0.05]))
        elif kind == "gate":
            case = _gate(_log(rng, 1, 65536), _log(rng, 256, 14336, 8), half, rng.random() < 0.3)
        else:
            case = _combine(_log(rng, 1, 8192), _log(rng, 512, 8192, 8), rng.randint(max(k, 4), 256), k, half, rng.random() < 0.5,
                            rng.choice([0.0, 0.0, 0.05]))
        if _cost(case) <= most[kind]:
            return case


def _picked(case, gen):
    """Distinct experts for every token, some of them more popular than others."""
    T, E, k = case["tokens"], case["experts"], case["k"]
    score = torch.rand((T, E), generator=gen, device="cuda") + 0.5 * torch.rand((1, E), generator=gen, device="cuda")
    picked = score.argsort(dim=1)[:, :k].to(torch.int32)
    if case.get("dropped"):
        picked = torch.where(torch.rand((T, k), generator=gen, device="cuda") < case["dropped"], torch.full_like(picked, -1), picked)
    return picked.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, st = case["kind"], {"case": case}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if kind == "route":
        st["logits"] = (1.5 * normal(case["tokens"], case["experts"])).to(_DT[case["dtype"]])
        st["bias"] = 0.1 * normal(case["experts"]) if case["bias"] else None
    elif kind == "blocks":
        st["experts"] = _picked(case, gen)
    elif kind == "gate":
        st["h"] = (2 * normal(case["rows"], 2 * case["width"])).to(_DT[case["dtype"]])
    else:
        picked, T, k, D = _picked(case, gen), case["tokens"], case["k"], case["width"]
        st["rows"] = _sorted_rows(picked, case["experts"])[1]
        if kind == "dispatch":
            st["x"] = (normal(T, D) * (0.5 + torch.rand((T, 1), generator=gen, device="cuda"))).to(_DT[case["dtype"]])
        else:
            st["y"] = normal(T * k, D).to(_DT[case["dtype"]])
            w = torch.rand((T, k), generator=gen, device="cuda") + 0.1
            st["weights"] = w / w.sum(1, keepdim=True)
            st["base"] = normal(T, D).to(_DT[case["dtype"]]) if case["base"] else None
    return st


def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    kind = case["kind"]
    if kind == "route":
        return _route_plain(st["logits"], st["bias"], case)
    if kind == "blocks":
        return _blocks_plain(st["experts"], case)
    if kind == "dispatch":
        return _dispatch_plain(st["x"], st["rows"], case)
    if kind == "gate":
        return _gate_plain(st["h"], case)
    return _combine_plain(st["y"], st["rows"], st["weights"], st["base"])


def _run_own(st, case):
    import tilelang_ascend_b200 as q
    kind = case["kind"]
    if kind == "route":
        return q.moe_route(st["logits"], case["k"], st["bias"], scoring=case["scoring"], num_groups=case["groups"],
                           top_groups=case["top_groups"], group_top=case["group_top"], renormalize=case["renormalize"], scale=case["scale"])
    if kind == "blocks":
        return q.moe_block_metadata(st["experts"], case["experts"], case["block"])
    if kind == "dispatch":
        return q.moe_act_quant(st["x"], st["rows"], case["round_scale"])
    if kind == "gate":
        return q.swiglu_act_quant(st["h"], case["round_scale"])
    return q.moe_combine(st["y"], st["rows"], st["weights"], st["base"])


# ---------------------------------------------------------------------------------------------- plain forms
def _route_plain(logits, bias, case):
    T, E, k, G = case["tokens"], case["experts"], case["k"], case["groups"]
    l = logits.double()
    if case["scoring"] == "softmax":
        e = torch.exp(l - l.max(dim=1, keepdim=True).values)
        s = e / e.sum(dim=1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-l))
    c = s if bias is None else s + bias.double()
    order = l if bias is None else c  # without a bias the logits are in the scores' order
    if G > 1:
        best = c.view(T, G, E // G).sort(dim=2, descending=True).values[:, :, :case["group_top"]].sum(dim=2)
        best = best.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        stays = torch.zeros((T, G), dtype=torch.bool, device=l.device).scatter(1, best, True)
        order = torch.where(stays.repeat_interleave(E // G, dim=1), order, torch.full_like(order, -math.inf))
    picked = order.sort(dim=1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, picked)
    if case["renormalize"]:
        w = w / w.sum(dim=1, keepdim=True)
    return (w * case["scale"]).float(), picked.to(torch.int32)


def _sorted_rows(experts, E):
    """(expert of every pick, E where it was dropped; the place of every pick in the stack; the picks in the stack's order)."""
    flat = experts.reshape(-1).long()
    flat = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E))
    order = flat.sort(stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    rows = torch.where(flat < E, place, -2 - place)
    return flat, rows.to(torch.int32).view(experts.shape), order


def _blocks_plain(experts, case):
    E, bm, R = case["experts"], case["block"], experts.numel()
    flat, rows, _ = _sorted_rows(experts, E)
    sizes = torch.zeros(E + 1, dtype=torch.long, device=flat.device).index_add(0, flat, torch.ones_like(flat))[:E]
    first, count = sizes.cumsum(0) - sizes, (sizes + bm - 1) // bm
    end = count.cumsum(0)
    n = min(E, R)
    i = torch.arange(n + (R - n) // bm, device=flat.device)
    g = (i[:, None] >= end[None, :]).sum(dim=1)
    there = g < E
    g = g.clamp(max=E - 1)
    done = (i - (end - count)[g]) * bm
    table = torch.stack([torch.where(there, g, torch.full_like(g, -1)), torch.where(there, first[g] + done, torch.full_like(g, R)),
                         torch.where(there, (sizes[g] - done).clamp(max=bm), torch.zeros_like(g))], dim=1)
    return table.to(torch.int32), rows, sizes.to(torch.int32)


def _pow2_ceil(s):
    """The power of two that is not below a positive s, from its exponent bits."""
    bits = s.view(torch.int32)
    return (((bits >> 23) + ((bits & 0x7FFFFF) != 0).int()) << 23).view(torch.float32)


def _dispatch_plain(x, rows, case):
    v = x.float()
    amax = v.abs().amax(dim=1, keepdim=True).clamp(min=1e-4)
    s = amax / torch.full_like(amax, 127)  # (by a tensor: a rounded quotient, not the product with a rounded reciprocal)
    s = _pow2_ceil(s) if case["round_scale"] else s
    q = (v / s).clamp(-127, 127).round().to(torch.int8)
    T, k = rows.shape
    y = torch.empty((T * k, x.shape[1]), dtype=torch.int8, device=x.device)
    scales = torch.empty((T * k, 1), dtype=torch.float32, device=x.device)
    at, token = rows.reshape(-1, 1).long(), torch.arange(T, device=x.device).repeat_interleave(k)
    to = torch.where(at >= 0, at, -2 - at).view(-1)  # a dropped pick's place is cleared
    y[to] = torch.where(at >= 0, q[token], torch.zeros_like(q[:1]))
    scales[to] = torch.where(at >= 0, s[token], torch.zeros_like(s[:1]))
    return y, scales


def _gate_plain(h, case):
    F = case["width"]
    g, u = h[:, :F].double(), h[:, F:].double()
    a = g / (1 + torch.exp(-g)) * u
    amax = a.abs().amax(dim=1, keepdim=True).clamp(min=1e-4)
    s = (amax / torch.full_like(amax, 127)).float()
    s = _pow2_ceil(s) if case["round_scale"] else s
    return (a / s.double()).round().clamp(-127, 127).to(torch.int8), s


def _combine_plain(y, rows, weights, base):
    T, k = rows.shape
    at = rows.reshape(-1).long()
    picked = y.float()[at.clamp(min=0)].view(T, k, -1)
    w = torch.where(rows >= 0, weights, torch.zeros_like(weights))
    out = (picked * w[:, :, None]).sum(dim=1)
    if base is not None:
        out = out + base.float()
    return out.to(y.dtype)


# -------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    """The definitions once more, by other steps: picks one after another, places by counting, rows by a gather."""
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _route_exact(st["logits"].double(), st["bias"], case)
    if kind == "blocks":
        return _blocks_exact(st["experts"].cpu().tolist(), case)
    if kind == "dispatch":
        x, rows = st["x"].double(), st["rows"].reshape(-1).long()
        top = x.abs().max(dim=1).values
        s = (torch.maximum(top, torch.tensor(1e-4, device=x.device).double()) / 127.0).float().double()
        if case["round_scale"]:
            s = torch.exp2(torch.ceil(torch.log2(s)))
        codes = torch.round((x / s[:, None]).float().double()).to(torch.int8)
        token = torch.full_like(rows, -1)
        there = torch.nonzero(rows >= 0).view(-1)
        token[rows[there]] = there // case["k"]
        none = token < 0
        return codes[token].masked_fill(none[:, None], 0), s[token][:, None].masked_fill(none[:, None], 0.0)
    if kind == "gate":
        g, u = st["h"].double().chunk(2, dim=1)
        a = g * torch.sigmoid(g) * u
        top = torch.maximum(a.max(dim=1).values, -a.min(dim=1).values)
        s = (torch.maximum(top, torch.tensor(1e-4, device=a.device).double()) / 127.0).float().double()
        if case["round_scale"]:
            s = torch.exp2(torch.ceil(torch.log2(s)))
        return torch.round(a / s[:, None]).to(torch.int8), s[:, None]
    out = st["base"].double() if st["base"] is not None else torch.zeros((case["tokens"], case["width"]), dtype=torch.float64, device="cuda")
    for j in range(case["k"]):
        at = st["rows"][:, j].long()
        t = torch.nonzero(at >= 0).view(-1)
        out[t] += st["weights"][t, j, None].double() * st["y"][at[t]].double()
    return out


def _route_exact(l, bias, case):
    T, E = l.shape
    G, n = case["groups"], case["experts"] // case["groups"]
    s = torch.sigmoid(l) if case["scoring"] == "sigmoid" else torch.exp(l - torch.logsumexp(l, dim=1, keepdim=True))
    c = s + bias.double() if bias is not None else s
    key = c.clone() if bias is not None else l.clone()
    if G > 1:
        left, value = c.reshape(T, G, n).clone(), 0.0
        for _ in range(min(case["group_top"], n)):
            top = left.max(dim=2, keepdim=True)
            value = value + top.values[:, :, 0]
            left = left.scatter(2, top.indices, -math.inf)
        out = torch.ones((T, G), dtype=torch.bool, device=l.device)
        for _ in range(case["top_groups"]):
            g = (value == value.max(dim=1, keepdim=True).values).int().argmax(dim=1, keepdim=True)
            out, value = out.scatter(1, g, False), value.scatter(1, g, -math.inf)
        key[out[:, :, None].expand(T, G, n).reshape(T, E)] = -math.inf
    picked = []
    for _ in range(case["k"]):
        e = (key == key.max(dim=1, keepdim=True).values).int().argmax(dim=1, keepdim=True)
        picked.append(e)
        key = key.scatter(1, e, -math.inf)
    picked = torch.cat(picked, dim=1)
    w = torch.gather(s, 1, picked)
    return w * (case["scale"] / w.sum(dim=1, keepdim=True) if case["renormalize"] else case["scale"]), picked.to(torch.int32)


def _blocks_exact(experts, case):
    E, bm = case["experts"], case["block"]
    mine = [[] for _ in range(E + 1)]
    for t, picks in enumerate(experts):
        for j, e in enumerate(picks):
            mine[e if 0 <= e < E else E].append((t, j))
    rows, table, at = [[0] * case["k"] for _ in experts], [], 0
    R = case["k"] * len(experts)
    for e, picks in enumerate(mine):
        if e < E:
            table += [[e, at + i, min(bm, len(picks) - i)] for i in range(0, len(picks), bm)]
        for t, j in picks:
            rows[t][j] = at if e < E else -2 - at
            at += 1
    n = min(E, R)
    table += [[-1, R, 0]] * (n + (R - n) // bm - len(table))
    return tuple(torch.tensor(v, dtype=torch.int32) for v in (table, rows, [len(m) for m in mine[:E]]))


def work(case):
    kind = case["kind"]
    if kind == "gate":
        M, F = case["rows"], case["width"]
        return {"bytes": 5 * M * F + 4 * M, "flops": 8 * M * F}
    T, E, k = case["tokens"], case["experts"], case["k"]
    R = T * k
    if kind == "route":
        return {"bytes": T * E * _BYTES[case["dtype"]] + (4 * E if case["bias"] else 0) + 8 * R, "flops": 4 * T * E}
    if kind == "blocks":
        n = min(E, R)
        return {"bytes": 8 * R + 12 * (n + (R - n) // case["block"]) + 4 * E, "flops": R}
    D = case["width"]
    if kind == "dispatch":
        return {"bytes": 2 * T * D + R * D + 8 * R, "flops": 3 * T * D}
    kept = int(R * (1 - case["dropped"]))
    return {"bytes": 2 * kept * D + 8 * R + (4 if case["base"] else 2) * T * D, "flops": 2 * kept * D}
