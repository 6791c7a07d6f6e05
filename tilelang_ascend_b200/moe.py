"""What a mixture-of-experts layer runs around the grouped W8A8 product, on the GPU from the router's logits on.

    weights, experts = moe_route(logits, top_k, bias, scoring="sigmoid", num_groups=8, top_groups=4)
    meta, rows, sizes = moe_block_metadata(experts, E)
    a, sa = moe_act_quant(x, rows)                                            # int8 rows in the experts' order
    h = grouped_quant_matmul(a, W_gate_up, meta, s_gate_up, sa, out_dtype="bfloat16")
    b, sb = swiglu_act_quant(h)
    y = grouped_quant_matmul(b, W_down, meta, s_down, sb, out_dtype="bfloat16")
    out = moe_combine(y, rows, weights)

The reference's grouped GEMM (examples/grouped_gemm/example_grouped_gemm_fwd.py:44-113) starts from rows that are sorted already and
from a table that the host has built (:147-166); its quantiser (examples/deepseek_v4/act_quant.py:33-92) writes a token once.
Nothing here is read back by the host, so the whole layer can be captured in a graph.  Shapes, types, devices and errors are
checked as in ``ops``: contiguous CUDA tensors on one device, else ``ValueError``.  Inference only: results carry no gradient.
"""
from __future__ import annotations

import torch

from . import _lib, ops
from .ops import _check_tensor, _ptr, _require_cuda, _stream_handle

_ROUTE_DT = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16, torch.float32: _lib.DT_F32}
_HALF_DT = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}
_SCORING = {"softmax": 0, "sigmoid": 1}
# The limits of include/qgemm.h.  Counts above them are refused before outputs of that size are allocated.
_MOST = {"top_k": 32, "num_experts": 1024, "block_M": 128, "num_groups": 32, "top_groups": 32, "group_top": 2}
_MAX_BLOCKS = 715827882


def _check_2d(t, idx, name, dtypes, device=None):
    _require_cuda(t, name)
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got {t.dim()}-D")
    if t.dtype not in dtypes:
        raise ValueError(f"Buffer dtype mismatch for parameter {name}: expected {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    _check_tensor(t, idx, name, t.dtype, None, t.device if device is None else device)


def _check_counts(**counts):
    for name, v in counts.items():
        if not isinstance(v, int) or v < 1:
            raise ValueError(f"{name} must be a positive integer, got {v!r}")
        if v > _MOST[name]:
            raise _lib.QGemmError(f"{name} must be 1 to {_MOST[name]}, got {v}")


def moe_route(logits, top_k, bias=None, scoring="softmax", num_groups=1, top_groups=1, group_top=2, renormalize=True, scale=1.0,
              stream=None):
    """Router logits [T, E] (float32 / bfloat16 / float16) -> (weights [T, top_k] float32, experts [T, top_k] int32).

    ``s = softmax(logits)`` or ``sigmoid(logits)`` (``scoring``); the ``top_k`` experts with the largest ``s + bias`` (``bias``: optional
    float32 [E], enters the choice only), best first, ties to the lower index.  With ``num_groups`` > 1 only experts of the
    ``top_groups`` best of that many equal runs of experts are eligible, a group being worth the sum of its ``group_top`` (1 or 2)
    largest ``s + bias``.  The weights are the chosen ``s``, divided by their sum if ``renormalize``, times ``scale``.

    An expert whose logit (or bias) is -inf is never chosen; where a token has fewer than ``top_k`` left, its last experts are
    -1 with weight 0 (a padding token: a row of -inf).  Mask by -inf: a finite bias far below the others gives the same picks, but more
    slowly.  A NaN logit counts as largest; its weight is NaN, and with softmax or ``renormalize`` so are all of its token's."""
    if stream is None and scoring in _SCORING:
        we = (ops._host or ops._native()).moe_route(logits, top_k, bias, _SCORING[scoring], num_groups, top_groups, group_top, renormalize, scale)
        if we is not None:
            return we
    lib = _lib.load()
    _check_2d(logits, 0, "logits", tuple(_ROUTE_DT))
    dev = logits.device
    T, E = logits.shape
    if bias is not None:
        _check_tensor(bias, 2, "bias", torch.float32, (E,), dev)
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be one of {sorted(_SCORING)}, got {scoring!r}")
    _check_counts(top_k=top_k, num_groups=num_groups, top_groups=top_groups, group_top=group_top)
    weights = torch.empty((T, top_k), dtype=torch.float32, device=dev)
    experts = torch.empty((T, top_k), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        rc = lib.qgemm_moe_route(logits.data_ptr(), _ptr(bias), weights.data_ptr(), experts.data_ptr(), T, E, top_k, num_groups,
                                 top_groups, group_top, _SCORING[scoring], 1 if renormalize else 0, float(scale),
                                 _ROUTE_DT[logits.dtype], _stream_handle(stream, dev))
    _lib.check(rc, "qgemm_moe_route")
    return weights, experts


def moe_block_metadata(experts, num_experts, block_M=128, stream=None):
    """Routed experts [T, top_k] int32 -> (block_metadata [blocks, 3], rows [T, top_k], sizes [num_experts]), all int32 on the GPU.

    The picks are stacked expert by expert, in their order in ``experts`` within one.  ``rows`` holds each pick's place in the stack,
    ``sizes`` the rows of every expert, and ``block_metadata`` what ``build_block_metadata(sizes, block_M)`` has, followed by entries
    ``(-1, T * top_k, 0)``, which the grouped product skips, up to the largest table that so many picks can need: the host
    does not learn the sizes.  A pick outside ``0 .. num_experts - 1`` (-1) is dropped: it takes a place behind all
    others, ``rows`` holds ``-2 - place``, and no block covers it."""
    if stream is None:
        tables = (ops._host or ops._native()).moe_blocks(experts, num_experts, block_M)
        if tables is not None:
            return tables
    lib = _lib.load()
    _check_2d(experts, 0, "experts", (torch.int32,))
    dev = experts.device
    _check_counts(num_experts=num_experts, block_M=block_M)
    E, bm, R = num_experts, block_M, experts.numel()
    blocks = lib.qgemm_moe_block_count(R, E, bm)
    if blocks > _MAX_BLOCKS:
        raise _lib.QGemmError(f"no more than {_MAX_BLOCKS} blocks, got {R} picks in blocks of {bm}")
    meta = torch.empty((blocks, 3), dtype=torch.int32, device=dev)
    rows = torch.empty(experts.shape, dtype=torch.int32, device=dev)
    sizes = torch.empty((E,), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        rc = lib.qgemm_moe_blocks(experts.data_ptr(), meta.data_ptr(), rows.data_ptr(), sizes.data_ptr(), R, E, bm, _stream_handle(stream, dev))
    _lib.check(rc, "qgemm_moe_blocks")
    return meta, rows, sizes


def moe_act_quant(x, rows, round_scale: bool = False, stream=None):
    """bf16 / f16 tokens [T, N] -> (int8 [T * top_k, N], fp32 scales [T * top_k, 1]) in the order of ``rows`` (``moe_block_metadata``).

    Each token is quantised as by ``act_quant``, bit for bit, and written to its ``top_k`` places: ``A`` and ``scale_a`` of
    ``grouped_quant_matmul``.  The places of dropped picks are cleared.  ``rows`` names no place twice; a place that it names not
    at all is left as allocated."""
    if stream is None:
        ys = (ops._host or ops._native()).moe_act_quant(x, rows, round_scale)
        if ys is not None:
            return ys
    lib = _lib.load()
    _check_2d(x, 0, "x", tuple(_HALF_DT))
    dev = x.device
    T, N = x.shape
    _check_2d(rows, 1, "rows", (torch.int32,), dev)
    if rows.shape[0] != T:
        raise ValueError(f"Static shape mismatch for parameter rows: expected ({T}, top_k), got {tuple(rows.shape)}")
    k = rows.shape[1]
    y = torch.empty((T * k, N), dtype=torch.int8, device=dev)
    s = torch.empty((T * k, 1), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        rc = lib.qgemm_moe_act_quant(x.data_ptr(), rows.data_ptr(), y.data_ptr(), s.data_ptr(), T, N, k, _HALF_DT[x.dtype],
                                     1 if round_scale else 0, _stream_handle(stream, dev))
    _lib.check(rc, "qgemm_moe_act_quant")
    return y, s


def swiglu_act_quant(x, round_scale: bool = False, stream=None):
    """bf16 / f16 ``x`` [M, 2 F] or [batch, seq, 2 F], gate columns first -> (int8 [.., F], fp32 scales [.., 1]).

    ``a = silu(gate) * up``; ``scale = max(max |a|, 1e-4) / 127`` in fp32 (a power of two not below it when ``round_scale``);
    ``y`` the integer nearest to ``a / scale``.  Both are those of the exact ``a``: no rounding of the product to 16 bits lies
    between, and values next to a border, or beyond what 32 bits hold, are decided in 64 bits.  A row with an infinity or a NaN, or whose
    scale is beyond float32, has no number for its scale and unspecified ``y``."""
    if stream is None:
        ys = (ops._host or ops._native()).swiglu_act_quant(x, round_scale)
        if ys is not None:
            return ys
    lib = _lib.load()
    _require_cuda(x, "x")
    dev = x.device
    if x.dim() not in (2, 3):
        raise ValueError(f"x must be 2-D or 3-D, got {x.dim()}-D")
    if x.dtype not in _HALF_DT:
        raise ValueError(f"x must be bfloat16 or float16, got {x.dtype}")
    _check_tensor(x, 0, "x", x.dtype, None, dev)
    if x.shape[-1] % 2:
        raise ValueError(f"the last dimension of x holds gate and up columns and must be even, got {x.shape[-1]}")
    F = x.shape[-1] // 2
    M = x.numel() // (2 * F) if F else 0
    y = torch.empty(tuple(x.shape[:-1]) + (F,), dtype=torch.int8, device=dev)
    s = torch.empty(tuple(x.shape[:-1]) + (1,), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        rc = lib.qgemm_swiglu_act_quant(x.data_ptr(), y.data_ptr(), s.data_ptr(), M, F, _HALF_DT[x.dtype], 1 if round_scale else 0,
                                        _stream_handle(stream, dev))
    _lib.check(rc, "qgemm_swiglu_act_quant")
    return y, s


def moe_combine(y, rows, weights, base=None, stream=None):
    """Experts' outputs [R, N] (bf16 / f16) -> [T, N]: ``base[t] + sum_j weights[t, j] * y[rows[t, j]]``.

    ``rows`` [T, top_k] int32 as from ``moe_block_metadata`` (an entry outside ``0 .. R - 1`` adds nothing), ``weights`` [T, top_k] float32,
    ``base`` optional [T, N] of the type of ``y`` (a shared expert's output, a residual).  Summed in fp32, ``j`` ascending,
    rounded once."""
    if stream is None:
        out = (ops._host or ops._native()).moe_combine(y, rows, weights, base)
        if out is not None:
            return out
    lib = _lib.load()
    _check_2d(y, 0, "y", tuple(_HALF_DT))
    dev = y.device
    R, N = y.shape
    _check_2d(rows, 1, "rows", (torch.int32,), dev)
    T, k = rows.shape
    _check_tensor(weights, 2, "weights", torch.float32, (T, k), dev)
    if base is not None:
        _check_tensor(base, 3, "base", y.dtype, (T, N), dev)
    out = torch.empty((T, N), dtype=y.dtype, device=dev)
    with torch.cuda.device(dev):
        rc = lib.qgemm_moe_combine(y.data_ptr(), rows.data_ptr(), weights.data_ptr(), _ptr(base), out.data_ptr(), R, T, N, k,
                                   _HALF_DT[y.dtype], _stream_handle(stream, dev))
    _lib.check(rc, "qgemm_moe_combine")
    return out
