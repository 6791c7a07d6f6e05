"""GPU tests of the mixture operators where fp32 does not settle the answer, and of calls at their limits, against plain 64-bit
implementations (oracle/moe_oracle.py).

Picks, codes and scales are equal.  Weights: relative 2^-20 as for ordinary logits (two ulp each of exp and two quotients, the
sum's roundings, the factor; the differences of the logits here are exact in fp32), and 1e-37 where a weight leaves fp32's normal range."""
import math

import pytest
import torch

import tilelang_ascend_b200 as q
from oracle import moe_oracle as mo
from oracle import qgemm_oracle as oc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(*seed):
    return torch.Generator().manual_seed(sum((i + 1) * 7919 * int(s) for i, s in enumerate(seed)) % (1 << 31))


def _check_route(logits, top_k, bias=None, **kw):
    w, e = q.moe_route(logits.cuda(), top_k, None if bias is None else bias.cuda(), **kw)
    w_ref, e_ref, _ = mo.route_ref(logits, top_k, bias, **kw)
    assert torch.equal(e.cpu(), e_ref)
    assert (w.cpu().double() - w_ref).abs().le(2.0 ** -20 * w_ref.abs() + 1e-37).all()
    return w, e


# ------------------------------------------------------------------------------------ routing: equal values at the last place
def _border_rows(T, E, k, copies, base, better, g):
    """Rows in which some experts are clearly above ``base``, ``copies`` of them are equal to it across the last place, and up to three
    at random places are ``better`` by less than fp32 scores (or shortened keys) show; all others are clearly below."""
    logits = base - 3.0 - torch.randint(0, 8, (T, E), generator=g).float()
    for t in range(T):
        order = torch.randperm(E, generator=g)
        above, late = int(torch.randint(0, k, (1,), generator=g)), 1 + t % 3
        logits[t, order[:above]] = base + 1.0
        logits[t, order[above:above + copies]] = base
        logits[t, order[above + copies:above + copies + late]] = better
    return logits


@pytest.mark.parametrize("E,k,copies", [(64, 1, 2), (64, 6, 7), (64, 4, 45), (256, 1, 2), (256, 8, 10), (256, 8, 60), (1024, 2, 3), (1024, 8, 9), (1024, 4, 100),
                                        (40, 32, 33), (513, 3, 5)])
@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_equal_logits_in_front_of_one_a_step_above(E, k, copies, groups, scoring):
    """fp32 logits without a bias: the places within a lane take the lowest bits of the keys, equal logits do not end the search."""
    if E % groups or E // groups < k:
        groups = 1
    base = torch.tensor(1.0)
    better = torch.nextafter(base, torch.tensor(2.0))
    logits = _border_rows(18, E, k, copies, float(base), float(better), _gen(E, k, copies))
    logits[0, 0] = logits[0, 1] = base
    logits[0, 2] = better
    _check_route(logits, k, scoring=scoring, num_groups=groups, top_groups=1, group_top=1)


@pytest.mark.parametrize("E,k,copies", [(64, 1, 2), (64, 6, 7), (64, 4, 45), (256, 8, 10), (256, 8, 60), (1024, 8, 9), (40, 32, 33), (513, 3, 5)])
@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("scoring,base,better,bias", [("sigmoid", 15.0, 15.0625, 0.0), ("sigmoid", 15.0, 15.0625, 1000.0), ("softmax", -20.0, -19.875, 0.0),
                                                      ("sigmoid", -18.0, -17.875, 0.25)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_route_equal_scores_in_front_of_a_near_one(E, k, copies, groups, scoring, base, better, bias, dt):
    """One bias for all, saturated or tiny scores: a tie of logits at the last place, and behind it one that only fp64 finds larger."""
    if E % groups or E // groups < k:
        groups = 1
    logits = _border_rows(12, E, k, copies, base, better, _gen(E, k, copies, groups))
    logits[:, -1] = 0.0 if scoring == "softmax" else base - 4.0
    assert torch.equal(logits.to(dt).float(), logits)
    _check_route(logits.to(dt), k, torch.full((E,), bias), scoring=scoring, num_groups=groups, top_groups=1, group_top=1)


# ---------------------------------------------------------------------------- routing: groups whose sums leave fp32's range
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_groups_of_huge_biases(scoring):
    """Two biases that fp32 holds and whose sum it does not: groups worth 6.0e38 and 6.4e38, and a group masked by fp32's lowest
    number beside one that offers nothing."""
    logits = torch.randn(6, 16, generator=_gen(1))
    bias = torch.zeros(16)
    bias[0:4], bias[8:12] = 3.0e38, 3.2e38
    _, e = _check_route(logits, 4, bias, scoring=scoring, num_groups=4, top_groups=1)
    assert ((e >= 8) & (e < 12)).all()
    bias = torch.full((16,), torch.finfo(F32).min)
    logits[:, :8] = -math.inf
    _, e = _check_route(logits, 3, bias, scoring=scoring, num_groups=2, top_groups=1)
    assert (e >= 8).all()
    logits[3:] = -math.inf
    _check_route(logits, 3, bias, scoring=scoring, num_groups=2, top_groups=1)


# --------------------------------------------------------------------------------------------- routing: weights of small scores
@pytest.mark.parametrize("picked", [(-29.0, -88.0), (-29.0, -88.0, -100.0), (0.0, -60.0), (-31.0, -90.0, -110.0), (-20.0, -29.5, -30.5, -95.0), (3.0, -31.0, -86.0),
                                    (90.0, -40.0), (-29.0, -29.0, -105.0), (-2000.0, -2001.0), (-5.0, -700.0)])
def test_route_sigmoid_weights_of_small_scores(picked):
    """Divided by their sum, scores that sigmoid takes out of fp32's range still have weights in it."""
    logits = torch.full((3, 64), -math.inf)
    for t in range(3):
        logits[t, torch.randperm(64, generator=_gen(t, len(picked)))[:len(picked)]] = torch.tensor(picked)
    _check_route(logits, len(picked), scoring="sigmoid")
    _check_route(logits, len(picked) + 2, scoring="sigmoid", scale=2.5)
    _check_route(logits, len(picked), scoring="sigmoid", renormalize=False)


# --------------------------------------------------------------------------------------- gate and quantise: bf16's whole range
def _far_rows(M, F, g):
    """Every third row has products that fp32 does not hold: gates below -87 beside ups of 1e29 and more, or products above 3.4e38."""
    x = torch.randn(M, 2 * F, generator=g) * 2
    for m in range(0, M, 3):
        kind, at = (m // 3) % 6, int(torch.randint(0, F, (1,), generator=g))
        if kind == 0:
            x[m, at], x[m, F + at] = -90.0, 1e38
        elif kind == 1:
            x[m] *= 1e18
            x[m, at] = x[m, F + at] = 1e20
        elif kind == 2:
            x[m, :F] = -87.0 - 15 * torch.rand(F, generator=g)
            x[m, F:] = torch.where(torch.rand(F, generator=g) < 0.5, 1e38, -1e38) * torch.rand(F, generator=g)
        elif kind == 3:
            x[m, at], x[m, F + at] = -87.5, 2.5e29
        elif kind == 4:
            x[m, :F], x[m, F:] = 1.5e19, torch.where(torch.rand(F, generator=g) < 0.5, 2e20, -2e20)
        else:
            x[m, at], x[m, F + at] = 3e30, -3e30  # 9e60 / 127: beyond fp32, the scale is an infinity
    return x.to(BF16)


@pytest.mark.parametrize("M,F", [(18, 8), (19, 264), (40, 2048), (20, 2056), (21, 4104), (18, 8200), (18, 16392), (18, 33000), (1500, 256), (3000, 2056), (1300, 7168)])
@pytest.mark.parametrize("round_scale", [False, True])
def test_gate_over_the_whole_range_of_bf16(M, F, round_scale):
    x = _far_rows(M, F, _gen(M, F))
    assert torch.isfinite(x.float()).all()
    y, s = [t.cpu() for t in q.swiglu_act_quant(x.cuda(), round_scale)]
    y_ref, s_ref = [t.cpu() for t in mo.swiglu_act_quant_ref(x.cuda(), round_scale)]
    there = torch.isfinite(mo.swiglu_act_quant_ref(x.cuda())[1].cpu()).view(-1)
    assert torch.equal(s[there], s_ref[there]) and torch.equal(y[there], y_ref[there])
    assert (s[~there] == math.inf).all() and int((~there).sum()) == len(range(15, M, 18))

@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("F", [264, 4104, 33000])
def test_gate_infinities_beside_far_products(value, F):
    """An infinity or a NaN among the inputs keeps the row's scale from being a number, whatever the others are."""
    x = _far_rows(24, F, _gen(F))
    want = [t.cpu() for t in q.swiglu_act_quant(x.cuda())]
    x[6, 3] = x[9, F + 7] = x[12, F - 1] = value
    y, s = [t.cpu() for t in q.swiglu_act_quant(x.cuda())]
    assert not torch.isfinite(s[[6, 9, 12]]).any()
    keep = [m for m in range(24) if m not in (6, 9, 12, 15)]
    assert torch.equal(y[keep], want[0][keep]) and torch.equal(s[keep], want[1][keep])


# ------------------------------------------------------------------- the grouped product over tables as long as the worst one
@pytest.mark.parametrize("sizes,K,N", [((300,), 272, 528), ((700, 513), 144, 2064), ((1000, 385, 257), 272, 4096), ((1,) * 16, 528, 4112), ((129,) * 11 + (81,), 400, 2048),
                                       ((0, 5, 0), 144, 272)])
@pytest.mark.parametrize("layout", ["KN", "NK"])
def test_grouped_product_over_host_built_tables_of_the_worst_length(sizes, K, N, layout):
    """Tables that the host built and that are as long as one made on the device: against the oracle, and with entries added."""
    g = torch.Generator(device="cuda").manual_seed(K + N)
    G, R = len(sizes), sum(sizes)
    A = torch.randint(-128, 128, (R, K), dtype=torch.int8, generator=g, device="cuda")
    B = torch.randint(-128, 128, (G, K, N) if layout == "KN" else (G, N, K), dtype=torch.int8, generator=g, device="cuda")
    s, sa = torch.rand((G, N), generator=g, device="cuda"), torch.rand(R, generator=g, device="cuda")
    table = q.build_block_metadata(sizes, 128)
    worst = min(R, G) + (R - min(R, G)) // 128
    if 0 not in sizes:
        assert len(table) == worst
    kw = dict(out_dtype=BF16, b_layout=layout)
    ref = torch.zeros(R, N, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(sizes):
        b = B[i].double() if layout == "KN" else B[i].double().t()
        ref[at:at + n] = (A[at:at + n].double() @ b).to(torch.int32)  # exact: below 2^53
        at += n
    got, acc = q.grouped_quant_matmul(A, B, table.cuda(), s, sa, return_accumulators=True, **kw)
    assert torch.equal(acc, ref)
    more = torch.cat([table, torch.tensor([[-1, R, 0]], dtype=torch.int32).repeat(worst, 1)]).cuda()
    assert torch.equal(q.grouped_quant_matmul(A, B, more, s, sa, **kw), got)
    assert torch.equal(q.grouped_quant_matmul(A, B, table.cuda(), s, sa, **kw), got)


@pytest.mark.parametrize("K,N,layout", [(144, 4096, "KN"), (272, 2048, "NK"), (16, 1040, "KN")])
def test_grouped_product_of_many_entries_per_cta(K, N, layout):
    """More items than 32 for every CTA, most of them without rows, in runs of any length."""
    g = _gen(K, N)
    sizes = [int(v) for v in torch.randint(0, 200, (64,), generator=g)]
    G, R = len(sizes), sum(sizes)
    A = torch.randint(-128, 128, (R, K), dtype=torch.int8, generator=g).cuda()
    B = torch.randint(-128, 128, (G, K, N) if layout == "KN" else (G, N, K), dtype=torch.int8, generator=g).cuda()
    s, sa = torch.rand((G, N), generator=g).cuda(), torch.rand(R, generator=g).cuda()
    used = q.build_block_metadata(sizes, 128)
    want = q.grouped_quant_matmul(A, B, used.cuda(), s, sa, out_dtype=BF16, b_layout=layout)
    none = torch.tensor([[-1, R, 0], [0, 0, 0], [3, R, 4]], dtype=torch.int32)
    for longest in (20, 300):
        pieces = []
        for entry in used:
            n = int(torch.randint(0, longest, (1,), generator=g))
            pieces += [none[torch.randint(0, 3, (n,), generator=g)], entry[None]]
        table = torch.cat(pieces + [none[:1].repeat(900, 1)])
        assert len(table) * ((N + 255) // 256) > 32 * 148
        got = q.grouped_quant_matmul(A, B, table.cuda(), s, sa, out_dtype=BF16, b_layout=layout)
        assert torch.equal(got, want)


# --------------------------------------------------------------------------------------------------------- limits of the counts
def test_counts_beyond_the_limits_are_refused_before_anything_is_allocated():
    l, e = torch.zeros((4, 64), device="cuda"), torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    held = torch.cuda.memory_reserved()
    for n in (1025, 10 ** 10, 10 ** 12, 2 ** 63, 2 ** 64 + 5, 10 ** 30):
        with pytest.raises(q.QGemmError):
            q.moe_block_metadata(e, n)
        with pytest.raises(q.QGemmError):
            q.moe_block_metadata(e, 4, block_M=n)
        with pytest.raises(q.QGemmError):
            q.moe_route(l, n)
        for name in ("num_groups", "top_groups", "group_top"):
            with pytest.raises(q.QGemmError):
                q.moe_route(l, 2, **{name: n})
        for kw in (dict(top_k=n), dict(top_k=2, num_groups=n), dict(top_k=2, group_top=2 ** 32 + 2)):
            with pytest.raises(q.QGemmError):
                q.moe_route(l, **kw, stream=torch.cuda.current_stream())
        with pytest.raises(q.QGemmError):
            q.moe_block_metadata(e, n, stream=torch.cuda.current_stream())
    assert torch.cuda.memory_reserved() <= held + (4 << 20)
