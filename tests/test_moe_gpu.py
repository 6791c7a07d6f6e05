"""GPU tests of the operators around the experts' products, against plain 64-bit implementations (oracle/moe_oracle.py).

Tolerances.  Picks, tables, places and int8 codes are equal.  Weights: exp and two quotients are good to 2 ulp (2 * 2^-24 each
half), the sum of up to 32 of them to 5 roundings, the factor to one, and exp's argument l - max is off by |l - max| 2^-24 at most: under 16 * 2^-24 =
2^-20, relative, for picks within a few units of the largest.  Combined rows: half a step of the output type, and
for the fp32 sum of top_k products and a base (top_k + 2) * 2^-24 of the sum of the absolute values."""
import math

import pytest
import torch

import tilelang_ascend_b200 as q
from oracle import moe_oracle as mo
from oracle import qgemm_oracle as oc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
WEIGHT_TOL = 2.0 ** -20


def _gen(*seed):
    return torch.Generator().manual_seed(sum((i + 1) * 7919 * int(s) for i, s in enumerate(seed)) % (1 << 31))


# ----------------------------------------------------------------------------------------------------- routing
def _check_route(logits, top_k, bias=None, **kw):
    w, e = q.moe_route(logits.cuda(), top_k, None if bias is None else bias.cuda(), **kw)
    w_ref, e_ref, _ = mo.route_ref(logits, top_k, bias, **kw)
    assert w.dtype == F32 and e.dtype == torch.int32 and w.shape == e.shape == (logits.shape[0], top_k)
    assert torch.equal(e.cpu(), e_ref)
    assert torch.equal(torch.isnan(w.cpu()), torch.isnan(w_ref))
    w, w_ref = torch.nan_to_num(w.cpu().double(), nan=0.0), torch.nan_to_num(w_ref, nan=0.0)
    assert (w - w_ref).abs().le(WEIGHT_TOL * w_ref.abs() + 1e-37).all()
    return w, e


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 256, 8), (3, 7, 7), (33, 32, 4), (5, 33, 2), (9, 60, 6), (130, 64, 8), (2, 129, 10), (17, 256, 1),
                                   (4, 257, 8), (6, 512, 32), (3, 513, 5), (2, 1024, 16)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("biased", [False, True])
def test_route_without_groups(T, E, k, scoring, dt, biased):
    g = _gen(T, E, k, biased)
    logits = (torch.randn(T, E, generator=g) * 2).to(dt)
    bias = torch.randn(E, generator=g) * 0.2 if biased else None
    _check_route(logits, k, bias, scoring=scoring, renormalize=k % 2 == 0, scale=1.0 if k % 3 else 2.5)


@pytest.mark.parametrize("E,groups,top_groups,k", [(256, 8, 4, 8), (60, 12, 5, 6), (64, 32, 3, 4), (36, 3, 2, 10), (160, 8, 3, 6), (1024, 4, 1, 32),
                                                   (16, 16, 5, 5), (20, 2, 2, 3), (384, 1, 1, 8), (10, 5, 1, 2), (992, 31, 30, 7)])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("scoring,biased,dt", [("sigmoid", True, F32), ("softmax", True, BF16), ("softmax", False, F32), ("sigmoid", False, BF16)])
def test_route_with_groups(E, groups, top_groups, k, group_top, scoring, biased, dt):
    g = _gen(E, groups, group_top, biased)
    logits = (torch.randn(19, E, generator=g) * 1.5).to(dt)
    bias = torch.randn(E, generator=g) * 0.1 if biased else None
    _check_route(logits, k, bias, scoring=scoring, num_groups=groups, top_groups=top_groups, group_top=group_top)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_ties_go_to_the_lowest_index(scoring, biased, groups):
    g = _gen(groups, biased)
    logits = torch.randint(-2, 3, (40, 48), generator=g).float()
    logits[0] = 0.0
    logits[1] = torch.where(torch.arange(48) % 3 == 0, torch.tensor(-0.0), torch.tensor(0.0))  # both zeros alike
    bias = torch.randint(0, 2, (48,), generator=g) * 0.25 if biased else None
    _, e = _check_route(logits, 6, bias, scoring=scoring, num_groups=groups, top_groups=max(1, groups // 2))
    if not biased and groups == 1:
        assert e[0].tolist() == e[1].tolist() == [0, 1, 2, 3, 4, 5]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,group_top", [(1, 2), (4, 2), (4, 1)])
def test_route_scores_that_fp32_cannot_tell_apart(scoring, groups, group_top):
    """The bias cancels the differences of the scores to within a few steps of fp32: most decisions are nearer than the error of an
    fp32 score."""
    g = _gen(groups, group_top)
    E = 64
    l = torch.randn(1, E, generator=g)
    s = (torch.softmax(l.double(), 1) if scoring == "softmax" else torch.sigmoid(l.double()))[0]
    bias = (0.75 - s).float()
    logits = torch.cat([l.expand(24, E), l.expand(24, E) + torch.randn(24, E, generator=g) * 1e-7])
    c = mo.route_ref(logits, 1, bias, scoring)[2]
    assert float((c - 0.75).abs().max()) < 1e-6 and len(set(c[0].tolist())) > 8
    _check_route(logits, 12, bias, scoring=scoring, num_groups=groups, top_groups=max(1, groups // 2), group_top=group_top)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups", [1, 5])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_route_masks(scoring, biased, groups, dt):
    """Rows that offer nothing, fewer than top_k, or the lowest number of the type in place of -inf."""
    g = _gen(groups, biased)
    E, k = 40, 6
    logits = torch.randn(12, E, generator=g).to(dt)
    bias = torch.randn(E, generator=g) * 0.1 if biased else None
    logits[0] = -math.inf
    logits[1] = -math.inf
    logits[1, 17] = -3.0
    logits[2, 3:] = -math.inf
    logits[3, ::2] = -math.inf
    logits[4] = torch.finfo(dt).min
    logits[5, 5:] = torch.finfo(dt).min
    logits[6, 8:] = -math.inf  # one group of eight is left
    logits[7] = 80.0           # both score functions at their largest
    logits[8] = -90.0
    logits[8, 3] = -85.0
    if biased:
        bias[4] = bias[18] = -math.inf
    w, e = _check_route(logits, k, bias, scoring=scoring, num_groups=groups, top_groups=(groups + 1) // 2)
    assert e[0].tolist() == [-1] * k and w[0].tolist() == [0.0] * k
    assert e[1].tolist() == [17] + [-1] * (k - 1) and w[1].tolist() == [1.0] + [0.0] * (k - 1)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_nan_and_infinity(scoring, biased):
    g = _gen(biased)
    logits = torch.randn(4, 24, generator=g)
    logits[0, 9] = math.nan
    logits[1, 20] = math.nan
    logits[1, 3] = -math.inf
    bias = torch.randn(24, generator=g) * 0.1 if biased else None
    w, e = q.moe_route(logits.cuda(), 3, None if bias is None else bias.cuda(), scoring=scoring, renormalize=True)
    assert torch.isnan(w[:2]).all() and torch.isfinite(w[2:]).all()  # seen, and in its own tokens only
    assert ((e >= 0) & (e < 24)).all()
    if scoring == "sigmoid" or not biased:
        assert int(e[0, 0]) == 9 and int(e[1, 0]) == 20
    logits[2, 11] = math.inf
    w, e = q.moe_route(logits.cuda(), 3, scoring="sigmoid", renormalize=False)
    assert int(e[2, 0]) == 11 and float(w[2, 0]) == 1.0


def test_route_many_tokens_and_none():
    """More tokens than one wave of warps; the rows are independent, so a slice gives the same bits."""
    g = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.randn(40011, 72, generator=g, device="cuda")
    bias = torch.randn(72, generator=g, device="cuda") * 0.1
    kw = dict(scoring="sigmoid", num_groups=6, top_groups=3)
    w, e = q.moe_route(logits, 5, bias, **kw)
    for a, b in ((0, 50), (39990, 40011)):
        w2, e2 = _check_route(logits[a:b].cpu(), 5, bias.cpu(), **kw)
        assert torch.equal(e[a:b], e2)
    w0, e0 = q.moe_route(logits[:0], 5, bias, **kw)
    assert w0.shape == e0.shape == (0, 5)
    assert torch.equal(q.moe_route(logits, 5, bias, **kw)[0], w)


def test_route_rejects():
    l = torch.zeros(4, 64, device="cuda")
    for kw in (dict(scoring="relu"), dict(num_groups=0), dict(top_groups=0), dict(bias=torch.zeros(63, device="cuda")),
               dict(bias=torch.zeros(64)), dict(bias=torch.zeros(64, device="cuda", dtype=F16)), dict(bias=torch.zeros(1, 64, device="cuda"))):
        with pytest.raises(ValueError):
            q.moe_route(l, 4, **kw)
    for bad in (l.t(), l.double(), l[0], l.view(1, 4, 64), l[:, :32]):
        with pytest.raises(ValueError):
            q.moe_route(bad, 4)
    for k in (0, -1, 2.0, None):
        with pytest.raises(ValueError):
            q.moe_route(l, k)
    for k, kw in ((33, {}), (9, dict(num_groups=8)), (4, dict(num_groups=7)), (4, dict(num_groups=8, top_groups=9)), (4, dict(group_top=3))):
        with pytest.raises(q.QGemmError):
            q.moe_route(l, k, **kw)
    with pytest.raises(q.QGemmError):
        q.moe_route(torch.zeros(2, 1025, device="cuda"), 1)
    with pytest.raises(q.QGemmError):
        q.moe_route(torch.zeros(2, 0, device="cuda"), 1)


# ------------------------------------------------------------------------------------------------- block tables
def _check_blocks(experts, E, bm):
    meta, rows, sizes = q.moe_block_metadata(experts.cuda(), E, bm)
    table, rows_ref, sizes_ref = mo.blocks_ref(experts, E, bm)
    assert meta.dtype == rows.dtype == sizes.dtype == torch.int32
    assert torch.equal(sizes.cpu(), sizes_ref) and torch.equal(rows.cpu(), rows_ref)
    n, R = len(table), experts.numel()
    assert meta.shape[0] >= n and meta.shape[1] == 3 and torch.equal(meta[:n].cpu(), table)
    assert torch.equal(meta[:n].cpu(), q.build_block_metadata(sizes_ref.tolist(), bm))
    assert meta[n:].cpu().tolist() == [[-1, R, 0]] * (len(meta) - n)
    return meta, rows, sizes


@pytest.mark.parametrize("T,k,E,bm", [(1, 1, 1, 128), (1, 8, 256, 128), (16, 8, 256, 128), (5, 2, 3, 1), (33, 4, 7, 2), (64, 8, 64, 64), (255, 1, 16, 100),
                                      (257, 8, 8, 128), (1000, 3, 1024, 128), (2049, 2, 100, 128), (4097, 5, 33, 64), (9001, 10, 384, 128)])
@pytest.mark.parametrize("dropped", [0.0, 0.2])
def test_blocks(T, k, E, bm, dropped):
    g = _gen(T, k, E)
    experts = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    bad = torch.tensor([-1, E, -(1 << 31), (1 << 31) - 1], dtype=torch.int32)[torch.randint(0, 4, (T, k), generator=g)]
    experts = torch.where(torch.rand(T, k, generator=g) < dropped, bad, experts)
    _check_blocks(experts, E, bm)


@pytest.mark.parametrize("T", [1, 31, 700, 5000, 70000])
def test_blocks_of_one_expert_and_of_none(T):
    _check_blocks(torch.full((T, 1), 2, dtype=torch.int32), 3, 128)
    _check_blocks(torch.full((T, 1), -1, dtype=torch.int32), 3, 128)
    _check_blocks(torch.arange(T, dtype=torch.int32).flip(0).view(T, 1) % 3, 3, 128)


def test_blocks_of_no_tokens_and_rejects():
    meta, rows, sizes = q.moe_block_metadata(torch.zeros((0, 4), dtype=torch.int32, device="cuda"), 5)
    assert meta.shape == (0, 3) and rows.shape == (0, 4) and sizes.tolist() == [0] * 5
    e = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    for bad in (e.long(), e.t(), e[0], e.view(1, 4, 2)):
        with pytest.raises(ValueError):
            q.moe_block_metadata(bad, 5)
    for kw in (dict(num_experts=0), dict(num_experts=-3), dict(num_experts=5, block_M=0), dict(num_experts=5.0)):
        with pytest.raises(ValueError):
            q.moe_block_metadata(e, **kw)
    for kw in (dict(num_experts=1025), dict(num_experts=5, block_M=129)):
        with pytest.raises(q.QGemmError):
            q.moe_block_metadata(e, **kw)


# ------------------------------------------------------------------------------------------- quantise into places
@pytest.mark.parametrize("T,N,k", [(1, 8, 1), (1, 7168, 8), (7, 264, 3), (33, 1024, 2), (130, 2048, 10), (16, 4104, 4), (5, 8200, 1), (3, 16392, 2), (2, 40000, 5),
                                   (700, 512, 6), (1201, 1032, 2)])
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("round_scale", [False, True])
def test_dispatch_is_the_quantiser_row_by_row(T, N, k, dt, round_scale):
    g = _gen(T, N, k)
    x = (torch.randn(T, N, generator=g) * torch.rand(T, 1, generator=g) * 8).to(dt)
    x[T // 2] = 0
    experts = torch.randint(-1, 6, (T, k), generator=g, dtype=torch.int32)
    rows = mo.blocks_ref(experts, 6, 128)[1]
    y, s = q.moe_act_quant(x.cuda(), rows.cuda(), round_scale)
    y1, s1 = oc.act_quant_torch_ref(x, round_scale)
    y_ref, s_ref = torch.zeros(T * k, N, dtype=torch.int8), torch.zeros(T * k, 1)
    for t in range(T):
        for j in range(k):
            if rows[t, j] >= 0:
                y_ref[rows[t, j]], s_ref[rows[t, j]] = y1[t], s1[t]
    assert torch.equal(s.cpu(), s_ref) and torch.equal(y.cpu(), y_ref)


def test_dispatch_places_outside_are_passed_over():
    """-1 and places behind the stack write nothing; what nobody names stays as it was (the C ABI writes into the caller's buffers)."""
    from tilelang_ascend_b200 import _lib
    lib = _lib.load()
    T, N, k = 3, 64, 2
    x = torch.randn(T, N, generator=_gen(1)).to(BF16).cuda()
    big = (1 << 31) - 1
    rows = torch.tensor([[4, -1], [6, big], [-(1 << 31), -2 - 6]], dtype=torch.int32, device="cuda")
    y = torch.full((T * k + 2, N), 77, dtype=torch.int8, device="cuda")
    s = torch.full((T * k + 2,), 5.0, device="cuda")
    assert lib.qgemm_moe_act_quant(x.data_ptr(), rows.data_ptr(), y.data_ptr(), s.data_ptr(), T, N, k, _lib.DT_BF16, 0,
                                   torch.cuda.current_stream().cuda_stream) == 0
    y1, s1 = q.act_quant(x)
    assert torch.equal(y[4], y1[0]) and float(s[4]) == float(s1[0])
    for r in (0, 1, 2, 3, 5, 6, 7):
        assert (y[r] == 77).all() and float(s[r]) == 5.0


def test_dispatch_empty_and_rejects():
    x, rows = torch.zeros((4, 64), dtype=BF16, device="cuda"), torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
    y, s = q.moe_act_quant(x[:0], rows[:0])
    assert y.shape == (0, 64) and s.shape == (0, 1)
    for a, r in ((x.float(), rows), (x.t(), rows), (x[0], rows), (x, rows.long()), (x, rows[:3]), (x, rows.t()), (x, rows.cpu()), (x, rows.view(-1))):
        with pytest.raises(ValueError):
            q.moe_act_quant(a, r)
    with pytest.raises(q.QGemmError):
        q.moe_act_quant(torch.zeros((4, 12), dtype=BF16, device="cuda"), rows)
    with pytest.raises(q.QGemmError):
        q.moe_act_quant(x, rows[:, :0].contiguous())
    with pytest.raises(q.QGemmError):  # an offset of half a row: not on a 16-byte boundary
        q.moe_act_quant(torch.zeros(4 * 64 + 4, dtype=BF16, device="cuda")[4:].view(4, 64), rows)


# ------------------------------------------------------------------------------------------- gate and quantise
def _check_gate(x, round_scale=False):
    y, s = q.swiglu_act_quant(x.cuda(), round_scale)
    y_ref, s_ref = mo.swiglu_act_quant_ref(x, round_scale)
    assert y.dtype == torch.int8 and s.dtype == F32 and y.shape == y_ref.shape and s.shape == s_ref.shape
    assert torch.equal(s.cpu(), s_ref) and torch.equal(y.cpu(), y_ref)
    return y, s


@pytest.mark.parametrize("M,F", [(1, 8), (1, 2048), (7, 264), (65, 256), (33, 520), (130, 1032), (16, 2056), (48, 4104), (5, 8192), (6, 8200), (2, 14336), (3, 33000),
                                 (1100, 136), (700, 2048)])
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("round_scale", [False, True])
def test_gate(M, F, dt, round_scale):
    g = _gen(M, F)
    x = (torch.randn(M, 2 * F, generator=g) * (0.1 + 4 * torch.rand(M, 1, generator=g))).to(dt)
    x[M // 2] = 0
    x[M - 1, F - 1], x[M - 1, 2 * F - 1] = 9.0, -30.0
    _check_gate(x, round_scale)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_gate_quotients_at_a_half(dt):
    """Equal gates, and ups that are simple fractions of the largest: quotients of n + 1/2 but for the rounding of the scale."""
    F = 1024
    x = torch.empty(64, 2 * F)
    for m in range(64):
        x[m, :F] = -3.0 + m / 8
        x[m, F:] = (torch.arange(F) % 255 - 127).float() * 0.5
    x[:, F] = 127.0
    x = x.to(dt)
    y, s = _check_gate(x)
    a = mo.swiglu_act_quant_ref(x)
    q64 = (lambda g, u: g / (1 + torch.exp(-g)) * u)(x[:, :F].double(), x[:, F:].double()) / a[1].double()
    assert ((q64 - q64.floor() - 0.5).abs() < 1e-4).float().mean() > 0.3  # the case is what it says


def test_gate_small_large_and_flat_rows():
    """Rows under the smallest scale, rows of equal magnitudes (every element a candidate for the largest), far gates."""
    F = 520
    g = _gen(3)
    x = torch.randn(8, 2 * F, generator=g)
    x[0] *= 1e-4
    x[1, :F], x[1, F:] = 1.0, torch.where(torch.rand(F, generator=g) < 0.5, 2.0, -2.0)
    x[2, :F] = -20.0 - 10 * torch.rand(F, generator=g)
    x[3, :F] = -40.0
    x[3, F:] = 1e9
    x[4, :F] = 100.0
    x[5, :F], x[5, F:] = 0.0, 5.0
    x[6] *= 1e8
    x[7, :F] = -1000.0
    for round_scale in (False, True):
        _check_gate(x.to(BF16), round_scale)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", [3, 300])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_gate_infinity_and_nan_stay_in_their_row(value, where, dt):
    F = 256
    x = torch.randn(5, 2 * F, generator=_gen(where)).to(dt)
    want = [t.clone() for t in mo.swiglu_act_quant_ref(x)]
    x[2, where] = value
    y, s = [t.cpu() for t in q.swiglu_act_quant(x.cuda())]
    assert not math.isfinite(float(s[2]))
    keep = [0, 1, 3, 4]
    assert torch.equal(y[keep], want[0][keep]) and torch.equal(s[keep], want[1][keep])


def test_gate_shapes_and_rejects():
    x = torch.randn(2, 3, 128, generator=_gen(9)).to(F16)
    y, s = _check_gate(x)
    assert y.shape == (2, 3, 64) and s.shape == (2, 3, 1)
    y, s = q.swiglu_act_quant(torch.zeros((0, 64), dtype=BF16, device="cuda"))
    assert y.shape == (0, 32) and s.shape == (0, 1)
    x = x.cuda()
    for bad in (x.float(), x.transpose(0, 1), x[0, 0], x[..., :127].contiguous(), x.view(2, 3, 2, 64)):
        with pytest.raises(ValueError):
            q.swiglu_act_quant(bad)
    for bad in (x[..., :40].contiguous(), x[..., :0].contiguous(), torch.zeros(4 * 64 + 4, dtype=BF16, device="cuda")[4:].view(4, 64)):
        with pytest.raises(q.QGemmError):
            q.swiglu_act_quant(bad)


# ----------------------------------------------------------------------------------------------------- combine
def _check_combine(y, rows, weights, base=None):
    out = q.moe_combine(y.cuda(), rows.cuda(), weights.cuda(), None if base is None else base.cuda())
    ref, size = mo.combine_ref(y, rows, weights, base)
    assert out.dtype == y.dtype and out.shape == ref.shape
    tol = torch.finfo(y.dtype).eps / 2 * ref.abs() + (rows.shape[1] + 2) * 2.0 ** -24 * size * 1.01 + torch.finfo(y.dtype).tiny * torch.finfo(y.dtype).eps
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    return out


@pytest.mark.parametrize("T,N,k", [(1, 8, 1), (1, 7168, 8), (3, 264, 2), (17, 1032, 3), (64, 2048, 6), (5, 4104, 10), (33, 16392, 4), (2, 40000, 8), (300, 512, 1), (3, 64, 32),
                                   (2, 72, 40)])
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("based", [False, True])
def test_combine(T, N, k, dt, based):
    g = _gen(T, N, k)
    rows = mo.blocks_ref(torch.randint(-1, 9, (T, k), generator=g, dtype=torch.int32), 9, 128)[1]
    y = torch.randn(T * k, N, generator=g).to(dt)
    w = torch.randn(T, k, generator=g)
    _check_combine(y, rows, w, torch.randn(T, N, generator=g).to(dt) if based else None)


def test_combine_rows_outside_twice_and_none():
    g = _gen(4)
    y = torch.randn(5, 24, generator=g).to(F16)
    y[3] = math.nan  # a row that nobody names
    big = (1 << 31) - 1
    rows = torch.tensor([[0, 0, 4], [-1, 5, 2], [big, -(1 << 31), -7], [1, -5, 1]], dtype=torch.int32)  # -2 - 3 = -5
    w = torch.randn(4, 3, generator=g)
    w[1, 0] = w[2, 1] = math.nan  # the weight of a dropped entry
    ref = mo.combine_ref(y, rows, torch.nan_to_num(w))[0]
    out = q.moe_combine(y.cuda(), rows.cuda(), w.cuda()).cpu()
    assert torch.isfinite(out).all() and (out[2] == 0).all() and torch.allclose(out.double(), ref, rtol=2e-3, atol=2e-3)
    base = torch.randn(4, 24, generator=g).to(F16)
    assert torch.equal(q.moe_combine(y.cuda(), rows.cuda(), w.cuda(), base.cuda())[2].cpu(), base[2])
    assert torch.equal(q.moe_combine(y[:0].cuda(), rows.cuda(), w.cuda(), base.cuda()).cpu(), base)
    assert q.moe_combine(y.cuda(), rows[:0].cuda(), w[:0].cuda()).shape == (0, 24)


def test_combine_onto_its_base():
    from tilelang_ascend_b200 import _lib
    g = _gen(6)
    y, base = torch.randn(12, 2056, generator=g).to(BF16).cuda(), torch.randn(6, 2056, generator=g).to(BF16).cuda()
    rows, w = torch.randperm(12, generator=g).to(torch.int32).view(6, 2).cuda(), torch.rand(6, 2, generator=g).cuda()
    want = q.moe_combine(y, rows, w, base)
    assert _lib.load().qgemm_moe_combine(y.data_ptr(), rows.data_ptr(), w.data_ptr(), base.data_ptr(), base.data_ptr(), 12, 6, 2056, 2, _lib.DT_BF16,
                                         torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(base, want)


def test_combine_rows_beyond_four_gigabytes():
    """The last rows of a stack of more than 2^32 bytes (and 2^31 values)."""
    R, N = 300000, 8192
    y = torch.empty((R, N), dtype=BF16, device="cuda")
    y[-2:] = torch.randn(2, N, generator=_gen(8)).to(BF16).cuda()
    y[0] = 1.0
    rows = torch.tensor([[R - 1, 0], [R - 2, R - 1]], dtype=torch.int32, device="cuda")
    w = torch.tensor([[1.0, 0.5], [0.25, -1.0]], device="cuda")
    out = q.moe_combine(y, rows, w)
    ref = torch.stack([y[-1].double() + 0.5, 0.25 * y[-2].double() - y[-1].double()])
    assert (out.double() - ref).abs().le(2.0 ** -8 * ref.abs() + 1e-6).all()


def test_combine_rejects():
    y, rows, w = torch.zeros((8, 64), dtype=BF16, device="cuda"), torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.zeros((4, 2), device="cuda")
    for args in ((y.float(), rows, w), (y.t(), rows, w), (y, rows.long(), w), (y, rows[:3], w), (y, rows, w.half()), (y, rows, w.cpu()),
                 (y, rows, w, y[:3]), (y, rows, w, y[:4].half()), (y, rows.view(-1), w.view(-1)), (y, rows, w, y[:4, :32])):
        with pytest.raises(ValueError):
            q.moe_combine(*args)
    with pytest.raises(q.QGemmError):
        q.moe_combine(torch.zeros((8, 12), dtype=BF16, device="cuda"), rows, w)
    with pytest.raises(q.QGemmError):
        q.moe_combine(y, rows[:, :0].contiguous(), w[:, :0].contiguous())


# ------------------------------------------------------------------------------------------------ the whole layer
def _layer(E, D, F, seed, dt=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")
    return dict(w1=torch.randint(-127, 128, (E, D, 2 * F), dtype=torch.int8, generator=g, device="cuda"), s1=(0.5 + rand(E, 2 * F)) * 1.5 / (73 * D ** 0.5),
                w2=torch.randint(-127, 128, (E, F, D), dtype=torch.int8, generator=g, device="cuda"), s2=(0.5 + rand(E, D)) * 2 / (73 * F ** 0.5),
                bias=rand(E) * 0.1)


def _run(p, x, logits, k, step=lambda: None, **kw):
    w, e = q.moe_route(logits, k, p["bias"], **kw)
    step()
    meta, rows, sizes = q.moe_block_metadata(e, p["w1"].shape[0])
    step()
    a, sa = q.moe_act_quant(x, rows)
    step()
    h = q.grouped_quant_matmul(a, p["w1"], meta, p["s1"], sa, out_dtype=x.dtype)
    step()
    b, sb = q.swiglu_act_quant(h)
    step()
    y = q.grouped_quant_matmul(b, p["w2"], meta, p["s2"], sb, out_dtype=x.dtype)
    step()
    return q.moe_combine(y, rows, w, x)


@pytest.mark.parametrize("T,E,D,F,k", [(1, 16, 256, 144, 4), (40, 8, 128, 64, 2), (300, 4, 256, 272, 3)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_layer_against_the_oracles(T, E, D, F, k, dt):
    """Route to combine as a layer runs it: every step but the last gives the oracle's bits for what it was given, so the whole is
    compared with the chain of oracles."""
    p = _layer(E, D, F, T)
    g = _gen(T, E)
    x, logits = torch.randn(T, D, generator=g).to(dt), torch.randn(T, E, generator=g)
    logits[T // 2] = -math.inf if T > 1 else 0.0  # a padding token
    kw = dict(scoring="sigmoid", num_groups=2, top_groups=1 if k <= E // 2 else 2)
    out = _run(p, x.cuda(), logits.cuda(), k, **kw).cpu()
    c = {n: t.cpu() for n, t in p.items()}
    w, e, _ = mo.route_ref(logits, k, c["bias"], **kw)
    table, rows, sizes = mo.blocks_ref(e, E, 128)
    a1, s1 = oc.act_quant_torch_ref(x)
    a, sa = torch.zeros(T * k, D, dtype=torch.int8), torch.zeros(T * k)
    for t in range(T):
        for j in range(k):
            if rows[t, j] >= 0:
                a[rows[t, j]], sa[rows[t, j]] = a1[t], s1[t, 0]
    h = oc.grouped_quant_matmul_ref(a, c["w1"], table, c["s1"], dt, scale_a=sa)
    b, sb = mo.swiglu_act_quant_ref(h)
    y = oc.grouped_quant_matmul_ref(b, c["w2"], table, c["s2"], dt, scale_a=sb.view(-1))
    ref, size = mo.combine_ref(y, rows, w, x)
    # a weight is off by 2^-20, the sum by (k + 2) * 2^-24, the result by half a step
    tol = torch.finfo(dt).eps / 2 * ref.abs() + (2.0 ** -20 + (k + 2) * 2.0 ** -24) * 1.01 * size + 1e-7
    assert ((out.double() - ref).abs() <= tol).all()
    assert float((ref - x.double()).abs().max()) > 0.1
    if T > 1:
        assert torch.equal(out[T // 2], x[T // 2])


@pytest.mark.parametrize("T,E,D,F,k", [(1, 64, 512, 256, 8), (24, 64, 1024, 512, 4), (700, 16, 512, 512, 4)])
def test_chain_of_layers(T, E, D, F, k):
    """All kernels of the layer are programmatic dependents of what is in front of them: layers behind one another, in buffers that the
    allocator hands out again at once, give the bits of the same layers with the device drained between the calls."""
    layers = [_layer(E, D, F, 10 + i) for i in range(3)]
    g = torch.Generator(device="cuda").manual_seed(T)
    x0 = torch.randn((T, D), generator=g, device="cuda").to(BF16)
    router = torch.randn((D, E), generator=g, device="cuda").to(BF16)

    def chain(step):
        x = x0
        for p in layers * 2:
            x = _run(p, x, x @ router / D ** 0.5, k, step, scoring="softmax", num_groups=8, top_groups=4)
            x = x / x.float().square().mean(1, keepdim=True).sqrt().to(BF16)
            step()
        return x

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert torch.equal(chain(lambda: None), want)
    assert torch.isfinite(want.float()).all() and not torch.equal(want, x0)


def test_layer_in_two_graphs_and_on_a_side_stream():
    """Captured once, replayed with other inputs; two graphs side by side on two streams; eager calls in between."""
    T, E, D, F, k = 48, 32, 512, 256, 4
    p = _layer(E, D, F, 3)
    kw = dict(scoring="sigmoid", num_groups=4, top_groups=2)

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        return torch.randn((T, D), generator=g, device="cuda").to(BF16), torch.randn((T, E), generator=g, device="cuda")

    want = [_run(p, *inputs(s), k, **kw) for s in range(6)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in range(6):
            assert torch.equal(_run(p, *inputs(s), k, **kw), want[s])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for s in range(2):
        x, l = inputs(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _run(p, x, l, k, **kw)
        graphs.append((graph, x, l, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        for i, (graph, x, l, out) in enumerate(graphs):
            x2, l2 = inputs(2 * turn + i)
            x.copy_(x2)
            l.copy_(l2)
        torch.cuda.synchronize()
        for (graph, x, l, out), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        assert torch.equal(_run(p, *inputs(5), k, **kw), want[5])
        torch.cuda.synchronize()
        for i, (graph, x, l, out) in enumerate(graphs):
            assert torch.equal(out, want[2 * turn + i])


def test_explicit_stream_arguments():
    T, E, D, k = 20, 16, 256, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    x, l = torch.randn((T, D), generator=g, device="cuda").to(F16), torch.randn((T, E), generator=g, device="cuda")
    w, e = q.moe_route(l, k)
    meta, rows, sizes = q.moe_block_metadata(e, E)
    a, sa = q.moe_act_quant(x, rows)
    b, sb = q.swiglu_act_quant(x)
    c = q.moe_combine(x.repeat(k, 1), rows, w, x)
    xs = x.repeat(k, 1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [*q.moe_route(l, k, stream=side), *q.moe_block_metadata(e, E, stream=side), *q.moe_act_quant(x, rows, stream=side),
           *q.swiglu_act_quant(x, stream=side.cuda_stream), q.moe_combine(xs, rows, w, x, stream=side)]
    side.synchronize()
    for u, v in zip(got, (w, e, meta, rows, sizes, a, sa, b, sb, c)):
        assert torch.equal(u, v)


def test_function_transforms_are_refused():
    x = torch.randn((2, 4, 64), device="cuda").half()
    rows = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    for call in (lambda t: q.moe_route(t, 2), lambda t: q.moe_act_quant(t, rows), q.swiglu_act_quant,
                 lambda t: q.moe_combine(t, rows, torch.zeros((4, 2), device="cuda"))):
        with pytest.raises(RuntimeError):
            torch.vmap(call)(x)


# 148 SMs: tiles of 128 columns in one round, of 256 in several rounds with a cut last one, of 256 in one round
@pytest.mark.parametrize("sizes,K,N", [((5, 0, 300, 1, 0, 0, 129, 2), 272, 528), ((700, 0, 1, 900, 128, 0, 640, 300, 0, 1100), 144, 2064),
                                       ((0, 0, 0, 0, 257), 1040, 256), ((64,) * 40, 512, 4096)])
@pytest.mark.parametrize("layout", ["KN", "NK"])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_grouped_product_passes_over_entries_without_rows(sizes, K, N, layout, dt):
    """Entries without rows behind the others, in front of them and between them change nothing: results, accumulators, rows that no
    block covers, and the calls behind."""
    g = torch.Generator(device="cuda").manual_seed(K + N)
    G, R = len(sizes), sum(sizes)
    A = torch.randint(-128, 128, (R + 9, K), dtype=torch.int8, generator=g, device="cuda")
    B = torch.randint(-128, 128, (G, K, N) if layout == "KN" else (G, N, K), dtype=torch.int8, generator=g, device="cuda")
    s, sa = torch.rand((G, N), generator=g, device="cuda"), torch.rand(R + 9, generator=g, device="cuda")
    used = q.build_block_metadata(sizes, 128)
    none = torch.tensor([[-1, R, 0], [0, 0, 0], [G, 0, 5], [0, R + 9, 5], [1, 3, -7]], dtype=torch.int32)
    most = G + (R + 9) // 128
    tables = [torch.cat([used, none[:1].repeat(most, 1)]), torch.cat([none.repeat(most, 1), used]),
              torch.cat([torch.cat([none, u[None]]) for u in used] + [none[:1].repeat(most, 1)])]
    kw = dict(out_dtype=dt, b_layout=layout)
    want, acc = q.grouped_quant_matmul(A, B, used.cuda(), s, sa, return_accumulators=True, **kw)
    for table in tables:
        got, got_acc = q.grouped_quant_matmul(A, B, table.cuda(), s, sa, return_accumulators=True, **kw)
        assert torch.equal(got, want) and torch.equal(got_acc, acc)
        assert torch.equal(q.grouped_quant_matmul(A, B, table.cuda(), s, sa, **kw), want)
        out = torch.full_like(want, 3.0)
        q.grouped_quant_matmul(A, B, table.cuda(), s, sa, out=out, **kw)
        assert torch.equal(out[:R], want[:R]) and (out[R:] == 3.0).all()
    empty = q.grouped_quant_matmul(A, B, none.repeat(most, 1).cuda(), s, sa, **kw)
    assert (empty == 0).all()


# ------------------------------------------------------------------------------------------- forms and their edges
# one, two, .. eight chunks per thread; rows shared by 32 .. 512 threads, full and one chunk over; few rows and more than the blocks
# that the SMs hold; rows that do not fit a thread's registers
GATE_FORMS = [(20000, 8), (20000, 256), (9000, 264), (7000, 512), (6000, 776), (5000, 1024), (5000, 1288), (5000, 1536), (4000, 1792),
              (4000, 2048), (3000, 2056), (2500, 3584), (2500, 4096), (1500, 4104), (1300, 7168), (1300, 8192), (700, 8200), (700, 14336), (400, 16392),
              (300, 28672), (200, 32776), (260, 256), (259, 2048), (258, 2056), (130, 4104), (65, 8200), (64, 16392)]


@pytest.mark.parametrize("M,F", GATE_FORMS)
@pytest.mark.parametrize("dt", [BF16, F16])
def test_gate_forms(M, F, dt):
    g = torch.Generator(device="cuda").manual_seed(M + F)
    x = (torch.randn((M, 2 * F), generator=g, device="cuda") * (0.5 + 3 * torch.rand((M, 1), generator=g, device="cuda"))).to(dt)
    for round_scale in (False, True):
        y, s = q.swiglu_act_quant(x, round_scale)
        y_ref, s_ref = mo.swiglu_act_quant_ref(x, round_scale)
        assert torch.equal(s, s_ref) and torch.equal(y, y_ref)


@pytest.mark.parametrize("T,N,k", [(9000, 8, 3), (9000, 256, 2), (9000, 264, 5), (5000, 520, 1), (4000, 1032, 2), (3000, 2056, 4), (2500, 4104, 2), (2000, 8200, 1),
                                   (1000, 16392, 2), (300, 32776, 3), (20, 7168, 40)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_dispatch_forms(T, N, k, dt):
    g = torch.Generator(device="cuda").manual_seed(T + N)
    x = torch.randn((T, N), generator=g, device="cuda").to(dt)
    rows = torch.randperm(T * k, generator=g, device="cuda").to(torch.int32).view(T, k)
    y1, s1 = q.act_quant(x)
    y, s = q.moe_act_quant(x, rows)
    at = rows.view(-1).long()
    assert torch.equal(y[at], y1.repeat_interleave(k, 0)) and torch.equal(s[at], s1.repeat_interleave(k, 0))


@pytest.mark.parametrize("R,E", [(128, 256), (129, 256), (128, 1024), (128, 1), (4096, 300), (4097, 300), (24576, 64), (24577, 64), (65536, 848), (65537, 848), (65537, 849),
                                 (70000, 1024), (131072, 256), (131073, 256), (300001, 40)])
def test_blocks_forms(R, E):
    g = torch.Generator(device="cuda").manual_seed(R + E)
    experts = torch.randint(-1, E, (R, 1), generator=g, device="cuda", dtype=torch.int32)
    experts[: R // 3] = torch.minimum(experts[: R // 3], torch.tensor(2, dtype=torch.int32, device="cuda"))  # some of them crowded
    meta, rows, sizes = q.moe_block_metadata(experts, E)
    flat = torch.where(experts.view(-1) < 0, E, experts.view(-1)).long()
    place = torch.empty(R, dtype=torch.int64, device="cuda")
    place[flat.sort(stable=True).indices] = torch.arange(R, device="cuda")
    assert torch.equal(rows.view(-1).long(), torch.where(flat < E, place, -2 - place))
    assert torch.equal(sizes.long(), torch.bincount(flat, minlength=E + 1)[:E])
    table = q.build_block_metadata(sizes.tolist())
    assert torch.equal(meta[: len(table)].cpu(), table) and (meta[len(table):, 2] == 0).all() and (meta[len(table):, 0] == -1).all()
    assert len(meta) == min(R, E) + (R - min(R, E)) // 128


@pytest.mark.parametrize("E,k,groups", [(64, 32, 1), (256, 32, 1), (1024, 32, 4), (40, 20, 2), (513, 9, 1), (512, 8, 16), (256, 3, 32)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_where_most_logits_are_equal(E, k, groups, biased):
    """More candidates than a warp has lanes: many equal values, and more picks than lanes that have one."""
    g = _gen(E, k, groups)
    logits = torch.randint(0, 2, (24, E), generator=g).float()
    logits[0] = 0.0
    logits[1] = 1.0
    logits[1, E // 2] = -math.inf
    logits[2, : E - k // 2] = -math.inf
    logits[3] = torch.randn(E, generator=g)
    bias = torch.zeros(E) if biased else None
    _check_route(logits, k, bias, scoring="sigmoid", num_groups=groups, top_groups=max(1, groups // 2))
    _check_route(logits, k, bias, scoring="softmax", num_groups=groups, top_groups=groups, renormalize=False)


@pytest.mark.parametrize("E,k", [(60, 4), (256, 8)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_route_of_slices(E, k, dt):
    """Logits that start off a 16-byte boundary are read one by one: the same picks."""
    g = torch.Generator(device="cuda").manual_seed(E)
    logits = torch.randn((41, E), generator=g, device="cuda").to(dt)
    shifted = torch.empty(41 * E + 1, dtype=dt, device="cuda")[1:].view(41, E)
    shifted.copy_(logits)
    for kw in (dict(), dict(bias=torch.randn(E, generator=g, device="cuda") * 0.1, scoring="sigmoid", num_groups=4, top_groups=2)):
        for a, b in zip(q.moe_route(logits, k, **kw), q.moe_route(shifted, k, **kw)):
            assert torch.equal(a, b)


def test_route_large_bias():
    """A bias far above the scores: c loses bits of the score, fp64 decides nearly everything."""
    g = _gen(77)
    logits = torch.randn(30, 64, generator=g)
    for scoring in ("softmax", "sigmoid"):
        _check_route(logits, 6, torch.full((64,), 1000.0), scoring=scoring)
        _check_route(logits, 6, torch.full((64,), -3e5) + torch.randint(0, 3, (64,), generator=g), scoring=scoring, num_groups=8, top_groups=3)


@pytest.mark.parametrize("E,groups,top_groups,k", [(160, 8, 3, 6), (348, 12, 7, 8), (1020, 17, 6, 8), (1023, 31, 30, 9), (1022, 7, 2, 16), (1000, 5, 3, 4), (90, 3, 1, 30),
                                                   (29, 29, 11, 11), (48, 24, 20, 3), (768, 16, 4, 10)])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("scoring,biased,dt", [("sigmoid", True, BF16), ("softmax", False, F16), ("softmax", True, F32)])
def test_route_groups_of_any_size(E, groups, top_groups, k, group_top, scoring, biased, dt):
    """Groups that fill their lanes in part, and lanes of up to 60 experts."""
    g = _gen(E, groups, group_top)
    logits = (torch.randn(11, E, generator=g) * 1.5).to(dt)
    logits[0, E // groups:] = -math.inf  # one group is left
    logits[1] = 0.25
    _check_route(logits, k, torch.randn(E, generator=g) * 0.1 if biased else None, scoring=scoring, num_groups=groups, top_groups=top_groups,
                 group_top=group_top)
