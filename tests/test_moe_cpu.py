"""CPU tests of the operators around the experts' products: what is refused before anything is launched, by the Python
layer and by the C ABI, the size of the block table, and the oracle against known answers."""
import ctypes
import math

import pytest
import torch

import tilelang_ascend_b200 as q
from oracle import moe_oracle as mo
from tilelang_ascend_b200 import _lib

SOME = ctypes.c_void_p(4096)  # a pointer that no refused call follows
ODD = ctypes.c_void_p(4097)


def _refused(rc, words):
    assert rc != 0 and words in _lib.last_error(), (rc, _lib.last_error())


def test_no_cpu_path():
    x, rows = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: q.moe_route(torch.zeros(4, 8), 2), lambda: q.moe_block_metadata(rows, 8), lambda: q.moe_act_quant(x, rows),
                 lambda: q.swiglu_act_quant(x), lambda: q.moe_combine(x, rows, torch.zeros(4, 2)), lambda: q.moe_route(None, 2),
                 lambda: q.swiglu_act_quant([1.0])):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


ROUTE = dict(logits=SOME, bias=None, weights=SOME, experts=SOME, T=4, E=64, k=4, groups=8, top_groups=4, group_top=2, scoring=0, renorm=1,
             scale=1.0, dt=_lib.DT_F32, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(T=-1), "tokens"), (dict(T=(1 << 30) + 1), "tokens"), (dict(E=0), "experts"), (dict(E=1025), "experts"), (dict(E=65), "num_groups"),
    (dict(groups=0), "num_groups"), (dict(groups=64), "num_groups"), (dict(top_groups=0), "top_groups"), (dict(top_groups=9), "top_groups"),
    (dict(k=0), "top_k"), (dict(k=33), "top_k"), (dict(k=9, top_groups=1), "top_k"), (dict(group_top=0), "group_top"),
    (dict(group_top=3), "group_top"), (dict(scoring=2), "scoring"), (dict(dt=_lib.DT_I32), "logits_dtype"), (dict(logits=None), "null"),
    (dict(weights=None), "null"), (dict(experts=None), "null"), (dict(logits=ODD), "aligned"), (dict(bias=ODD), "aligned")])
def test_route_refusals(change, words):
    _refused(_lib.load().qgemm_moe_route(*{**ROUTE, **change}.values()), words)


def test_route_of_no_tokens_needs_no_device():
    assert _lib.load().qgemm_moe_route(*{**ROUTE, "T": 0, "logits": None, "weights": None, "experts": None}.values()) == 0


BLOCKS = dict(experts=SOME, meta=SOME, rows=SOME, sizes=SOME, entries=8, E=8, block_M=128, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(entries=-1), "entries"), (dict(entries=(1 << 30) + 1), "entries"), (dict(E=0), "experts"), (dict(E=1025), "experts"),
    (dict(block_M=0), "block_M"), (dict(block_M=129), "block_M"), (dict(experts=None), "null"), (dict(meta=None), "null"), (dict(rows=None), "null"),
    (dict(sizes=None), "null"), (dict(sizes=None, entries=0), "null"), (dict(rows=ODD), "aligned")])
def test_blocks_refusals(change, words):
    _refused(_lib.load().qgemm_moe_blocks(*{**BLOCKS, **change}.values()), words)


QUANT = dict(X=SOME, rows=SOME, Y=SOME, S=SOME, T=4, N=64, k=2, dt=_lib.DT_BF16, round=0, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(T=-1), "T >= 0"), (dict(N=0), "multiple of 8"), (dict(N=12), "multiple of 8"), (dict(N=(1 << 30) + 8), "too large"), (dict(k=0), "top_k"),
    (dict(T=1 << 29, k=4), "2^30"), (dict(dt=_lib.DT_F32), "x_dtype"), (dict(X=None), "null"), (dict(rows=None), "null"), (dict(Y=None), "null"),
    (dict(S=None), "null"), (dict(X=ctypes.c_void_p(4104)), "16-byte"), (dict(Y=ctypes.c_void_p(4100)), "8-byte"), (dict(rows=ODD), "4-byte")])
def test_dispatch_refusals(change, words):
    _refused(_lib.load().qgemm_moe_act_quant(*{**QUANT, **change}.values()), words)


GATE = dict(X=SOME, Y=SOME, S=SOME, M=4, F=64, dt=_lib.DT_F16, round=0, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(M=-1), "M >= 0"), (dict(F=0), "multiple of 8"), (dict(F=20), "multiple of 8"), (dict(F=(1 << 29) + 8), "too large"),
    (dict(dt=_lib.DT_I32), "x_dtype"), (dict(X=None), "null"), (dict(Y=None), "null"), (dict(S=None), "null"),
    (dict(X=ctypes.c_void_p(4104)), "16-byte"), (dict(Y=ctypes.c_void_p(4100)), "8-byte"), (dict(S=ODD), "4-byte")])
def test_gate_refusals(change, words):
    _refused(_lib.load().qgemm_swiglu_act_quant(*{**GATE, **change}.values()), words)


COMBINE = dict(Y=SOME, rows=SOME, weights=SOME, base=None, out=SOME, R=8, T=4, N=64, k=2, dt=_lib.DT_BF16, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(T=-1), "T, R >= 0"), (dict(R=-1), "T, R >= 0"), (dict(N=0), "multiple of 8"), (dict(N=12), "multiple of 8"), (dict(N=(1 << 30) + 8), "too large"),
    (dict(k=0), "top_k"), (dict(T=1 << 29, k=4), "2^30"), (dict(dt=_lib.DT_F32), "dtype"), (dict(Y=None), "null"), (dict(rows=None), "null"),
    (dict(weights=None), "null"), (dict(out=None), "null"), (dict(Y=ctypes.c_void_p(4104)), "16-byte"), (dict(base=ctypes.c_void_p(4104)), "16-byte"),
    (dict(out=ctypes.c_void_p(4104)), "16-byte"), (dict(weights=ODD), "4-byte")])
def test_combine_refusals(change, words):
    _refused(_lib.load().qgemm_moe_combine(*{**COMBINE, **change}.values()), words)


@pytest.mark.parametrize("entries,experts,bm", [(0, 4, 128), (1, 4, 128), (3, 4, 128), (4, 4, 1), (5, 4, 2), (300, 3, 128), (129, 1, 128)])
def test_block_count_is_what_the_worst_sizes_need(entries, experts, bm):
    def most(rows, groups):  # the largest number of blocks over all sizes
        if groups == 1 or rows == 0:
            return -(-rows // bm)
        return max(-(-a // bm) + most(rows - a, groups - 1) for a in {0, 1, rows} if a <= rows)
    assert _lib.load().qgemm_moe_block_count(entries, experts, bm) == most(entries, experts)


def test_oracle_known_answers():
    l = torch.tensor([[0.0, math.log(3.0), 0.0, -math.inf]])
    w, e, _ = mo.route_ref(l, 2, renormalize=False)
    assert e.tolist() == [[1, 0]] and torch.allclose(w, torch.tensor([[0.6, 0.2]], dtype=torch.float64))
    w, e, _ = mo.route_ref(l, 4, scale=2.0)
    assert e.tolist() == [[1, 0, 2, -1]] and torch.allclose(w, torch.tensor([[1.2, 0.4, 0.4, 0.0]], dtype=torch.float64))
    # the groups {0, 1} and {2, 3}: by their two best 0.5 + 0.5 against 0.9 + 0, by their best the other way round
    b = torch.tensor([0.0, 0.0, 0.4, -0.5])
    z = torch.zeros(1, 4)
    assert mo.route_ref(z, 1, b, "sigmoid", 2, 1, 2)[1].tolist() == [[0]]
    assert mo.route_ref(z, 1, b, "sigmoid", 2, 1, 1)[1].tolist() == [[2]]
    table, rows, sizes = mo.blocks_ref(torch.tensor([[2, 0], [2, -1], [0, 2]], dtype=torch.int32), 3, 2)
    assert table.tolist() == [[0, 0, 2], [2, 2, 2], [2, 4, 1]] and sizes.tolist() == [2, 0, 3]
    assert rows.tolist() == [[2, 0], [3, -7], [1, 4]]
    y, s = mo.swiglu_act_quant_ref(torch.tensor([[0.0, 20.0, 1.0, 2.0]]))
    assert y.tolist() == [[0, 127]] and float(s[0]) == pytest.approx(40.0 / 127)
    out, size = mo.combine_ref(torch.tensor([[1.0], [2.0]]), torch.tensor([[0, 1], [1, -2]]), torch.tensor([[0.5, -1.0], [2.0, 9.0]]))
    assert out.tolist() == [[-1.5], [4.0]] and size.tolist() == [[2.5], [4.0]]
