"""Operators that stand around the expert layer in a transformer block: the norms with the
block's gate and residual sum, the choice of experts, and linear layers in 8-bit integers.

Like ``run``, they check their arguments (:class:`MoEArgumentError`), run on the current CUDA
stream without a host synchronisation, and compute in the hand-written CUDA of
``libmoe_b200.so``; there is no CPU or PyTorch path.  Tensors are ``[rows, cols]`` with adjacent
elements in a row; rows may be further apart than their length (slices of wider tensors).
The backward functions are explicit: they take what the forward took and the gradients of its
results.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _native

_TYPES = {torch.bfloat16: _native.BF16, torch.float16: _native.FP16, torch.float32: _native.FP32,
          torch.float8_e4m3fn: _native.E4M3, torch.int8: _native.INT8}
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


class MoEArgumentError(AssertionError, ValueError):
    """An input violates the definition of the layer or of the operator."""


def _check(cond: bool, msg: str):
    if not cond:
        raise MoEArgumentError(msg)


class BlockNormOut(NamedTuple):
    residual: torch.Tensor            # r', the residual stream behind the block
    x: torch.Tensor | None            # its norm (None without pre_weight)
    x_scale: torch.Tensor | None      # [ceil(cols / 128), rows] for an e4m3 x


class BlockNormGrads(NamedTuple):
    residual: torch.Tensor
    y: torch.Tensor | None
    pre_weight: torch.Tensor | None   # fp32
    post_weight: torch.Tensor | None  # fp32
    gate: torch.Tensor | None         # the gate's shape


class Selection(NamedTuple):
    idx: torch.Tensor                 # int32 [T, top_k], ascending; -1: no expert left
    w: torch.Tensor                   # float32 [T, top_k]
    counts: torch.Tensor | None       # int32 [E]


def _rows(t, name: str, shape=None, dtypes=_FLOATS, dev=None):
    """Checks a [rows, cols] tensor of the call; returns it."""
    _check(t.dim() == 2 and (t.shape[1] < 2 or t.stride(1) == 1),
           f"{name} must be [rows, cols] with adjacent elements in a row")
    _check(t.shape[0] < 2 or t.stride(0) >= 0, f"{name}: negative row stride")
    if shape is not None:
        _check(t.shape == shape, f"{name} must be {list(shape)}")
    _check(t.dtype in dtypes, f"{name} has an unsupported type {t.dtype}")
    _check(t.is_cuda, "all tensors must be CUDA tensors (there is no CPU path)")
    if dev is not None:
        _check(t.device == dev, "all tensors must be on one device")
    return t


def _result(t, name: str, shape, dtypes, dev):
    """Checks a tensor that receives a result: rows may not overlap."""
    _rows(t, name, shape, dtypes, dev)
    _check(shape[0] < 2 or t.stride(0) >= shape[1], f"{name}: rows overlap")
    return t


def _vector(t, name: str, n: int, dtypes, dev):
    if t is not None:
        _check(t.dim() == 1 and t.shape[0] == n and t.is_contiguous(), f"{name} must be a contiguous [{n}] tensor")
        _check(t.dtype in dtypes, f"{name} has an unsupported type {t.dtype}")
        _check(t.device == dev, "all tensors must be on one device")
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _type(t) -> int:
    return 0 if t is None else _TYPES[t.dtype]


def _ld(t) -> int:
    """Row pitch in elements (a single row's stride is arbitrary and says nothing)."""
    return 0 if t is None else t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _stream(dev) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _done(rc: int, what: str):
    if rc == _native.OK:
        return
    if rc == _native.ERR_ARG:
        raise MoEArgumentError(f"{what}: {_native.last_error()}")
    raise RuntimeError(f"{what} failed ({rc}): {_native.last_error()}")


def _gate_layout(gate, rows: int, cols: int, dev):
    """(row stride, varies along a row) of a gate [cols], [1, cols], [rows, 1], [1, 1] or [rows, cols]."""
    if gate is None:
        return 0, 0
    _check(gate.dtype in _FLOATS, f"gate has an unsupported type {gate.dtype}")
    _check(gate.device == dev, "all tensors must be on one device")
    g = gate.unsqueeze(0) if gate.dim() == 1 else gate
    _check(g.dim() == 2 and g.shape[0] in (1, rows) and g.shape[1] in (1, cols),
           "gate must be broadcastable to [rows, cols]")
    per_column = cols > 1 and g.shape[1] == cols
    per_row = rows > 1 and g.shape[0] == rows
    _check(not per_column or g.stride(1) == 1, "gate must have adjacent elements in a row")
    _check(not per_row or g.stride(0) > 0, "gate: pass a broadcast gate with its own size, not expanded")
    return g.stride(0) if per_row else 0, int(per_column)


@torch.no_grad()
def block_norm(y: torch.Tensor | None, residual: torch.Tensor | None, *, post_weight: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, scale: float = 1.0, pre_weight: torch.Tensor | None = None,
               eps: float = 1e-6, weight_offset: float = 0.0, x_dtype: torch.dtype | None = None,
               residual_out: torch.Tensor | None = None, out: torch.Tensor | None = None) -> BlockNormOut:
    """The end of one block and the beginning of the next, in one pass::

        n  = rms_norm(y) * (post_weight + weight_offset)      (n = y without post_weight)
        r' = residual + scale * gate * n
        x  = rms_norm(r') * (pre_weight + weight_offset)      (no x without pre_weight)

    ``y`` [rows, cols] is the block's output (None: x is the norm of ``residual``), ``residual``
    has y's type or fp32 (None: 0), ``gate`` is [cols], [1, cols], [rows, 1], [1, 1] or [rows, cols].
    ``x_dtype`` is the type of x (y's by default); ``torch.float8_e4m3fn`` quantises x per row and
    128 columns and returns ``x_scale`` [ceil(cols / 128), rows]: the ``hidden_states`` and
    ``hidden_states_scale`` of :func:`moe_swarm_b200.run`.  ``residual_out`` (may be ``residual``)
    and ``out`` receive r' and x instead of new tensors.
    """
    first = y if y is not None else residual
    _check(first is not None, "y or residual is required")
    _rows(first, "y" if y is not None else "residual")
    shape, dev = first.shape, first.device
    rows, cols = shape
    if y is not None and residual is not None:
        _rows(residual, "residual", shape, (y.dtype, torch.float32), dev)
    _vector(post_weight, "post_weight", cols, _FLOATS, dev)
    _vector(pre_weight, "pre_weight", cols, _FLOATS, dev)
    gate_ld, gate_cols = _gate_layout(gate, rows, cols, dev)
    r_dtype = residual.dtype if residual is not None else y.dtype
    if y is None:
        _check(residual_out is None, "residual_out is the residual itself without y")
    elif residual_out is None:
        residual_out = torch.empty(shape, dtype=r_dtype, device=dev)
    else:
        _result(residual_out, "residual_out", shape, (r_dtype,), dev)
    x = x_scale = None
    if pre_weight is not None:
        x_dtype = (out.dtype if out is not None else first.dtype) if x_dtype is None else x_dtype
        _check(x_dtype in _TYPES and x_dtype != torch.int8, f"unsupported x_dtype {x_dtype}")
        x = torch.empty(shape, dtype=x_dtype, device=dev) if out is None else _result(out, "out", shape, (x_dtype,), dev)
        if x_dtype == torch.float8_e4m3fn:
            x_scale = torch.empty(((cols + 127) // 128, rows), dtype=torch.float32, device=dev)
    a = _native.NormArgs(
        _ptr(y), _ptr(residual), _ptr(post_weight), _ptr(pre_weight), _ptr(gate), _ptr(residual_out), _ptr(x),
        _ptr(x_scale), _ld(y), _ld(residual), _ld(residual_out), _ld(x), gate_ld, rows, cols, _type(first),
        _TYPES[r_dtype], _type(post_weight), _type(pre_weight), _type(gate), _type(x), gate_cols, scale, eps,
        weight_offset)
    _done(_native.lib().moe_b200_block_norm(ctypes.byref(a), _stream(dev)), "block_norm")
    return BlockNormOut(residual if y is None else residual_out, x, x_scale)


@torch.no_grad()
def block_norm_backward(dx: torch.Tensor | None, dresidual: torch.Tensor | None, residual: torch.Tensor,
                        y: torch.Tensor | None, *, post_weight: torch.Tensor | None = None,
                        gate: torch.Tensor | None = None, scale: float = 1.0,
                        pre_weight: torch.Tensor | None = None, eps: float = 1e-6,
                        weight_offset: float = 0.0) -> BlockNormGrads:
    """Gradients of :func:`block_norm` from those of x (``dx``) and of r' (``dresidual``), either
    of which may be None.  ``residual`` is the forward's result r'; the other arguments are the
    forward's own.  With an e4m3 x, ``dx`` is the gradient of the values it stands for.

    Weight gradients are fp32.  The gate's gradient has the gate's shape, summed over what it is
    broadcast over: fp32 where it is summed, the gate's type for a [rows, cols] gate.
    """
    _rows(residual, "residual")
    shape, dev = residual.shape, residual.device
    rows, cols = shape
    given = y if y is not None else dx if dx is not None else residual
    _check(residual.dtype in (given.dtype, torch.float32), "residual must have y's type or fp32")
    _check(dx is not None or dresidual is not None, "dx or dresidual is required")
    _check(dx is None or pre_weight is not None, "dx needs pre_weight")
    _check(y is not None or (post_weight is None and gate is None), "post_weight and gate need y")
    for t, name, dtype in ((y, "y", given.dtype), (dx, "dx", given.dtype), (dresidual, "dresidual", residual.dtype)):
        if t is not None:
            _rows(t, name, shape, (dtype,), dev)
    _vector(post_weight, "post_weight", cols, _FLOATS, dev)
    _vector(pre_weight, "pre_weight", cols, _FLOATS, dev)
    gate_ld, gate_cols = _gate_layout(gate, rows, cols, dev)

    def new(like, dtype=None):
        return None if like is None else torch.empty(like.shape, dtype=dtype or like.dtype, device=dev)

    dres, dy = new(residual), new(y)
    dpre = new(pre_weight, torch.float32) if dx is not None else None
    dpost = new(post_weight, torch.float32)
    dgate = new(gate, None if gate_ld and gate_cols else torch.float32)
    lib = _native.lib()
    n = lib.moe_b200_block_norm_backward_workspace_size(rows, cols)
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=dev)
    a = _native.NormBackwardArgs(
        _ptr(dx), _ptr(dresidual), _ptr(residual), _ptr(y), _ptr(post_weight), _ptr(pre_weight), _ptr(gate),
        _ptr(dres), _ptr(dy), _ptr(dpre), _ptr(dpost), _ptr(dgate), _ld(dx), _ld(dresidual), _ld(residual), _ld(y),
        gate_ld, _ld(dres), _ld(dy), cols, rows, cols, _TYPES[given.dtype], _type(residual), _type(post_weight),
        _type(pre_weight), _type(gate), gate_cols, scale, eps, weight_offset)
    _done(lib.moe_b200_block_norm_backward(ctypes.byref(a), ws.data_ptr(), ws.numel(), _stream(dev)),
          "block_norm_backward")
    return BlockNormGrads(dres, dy, dpre, dpost, dgate)


_SCORES = {"sigmoid": 0, "softmax": 1}
_GROUP_SCORES = {"top2": 0, "max": 1}


@torch.no_grad()
def select_experts(logits: torch.Tensor, top_k: int, *, score: str = "sigmoid", bias: torch.Tensor | None = None,
                   n_group: int = 1, topk_group: int = 1, group_score: str = "top2", renormalize: bool = True,
                   scale: float = 1.0, counts: bool = False) -> Selection:
    """The ``top_k`` experts of each token and their weights, from router logits [T, E], E <= 512.

    ``score`` is "sigmoid" or "softmax"; ``bias`` [E] is added to the scores for the choice only.
    With ``n_group`` > 1 the experts form that many consecutive groups, scored by the sum of their
    two highest (biased) scores ("top2") or their highest ("max"), and only the ``topk_group``
    best are chosen from.  Ids come in ascending order (equal scores go to the lower id); the
    weights are the scores, divided by their sum if ``renormalize``, times ``scale``.  A logit of
    -inf or of its type's lowest value switches its expert off; slots left over hold id -1 and
    weight 0.  A row with a NaN score has ids -1 and NaN weights.  ``counts`` also returns how many
    tokens chose each expert.  idx and w are what :func:`moe_swarm_b200.run_routed` takes.
    """
    _rows(logits, "logits")
    T, E = logits.shape
    dev = logits.device
    _check(score in _SCORES, "score must be 'sigmoid' or 'softmax'")
    _check(group_score in _GROUP_SCORES, "group_score must be 'top2' or 'max'")
    _check(1 <= top_k <= E, "top_k must be in [1, number of experts]")
    _vector(bias, "bias", E, _FLOATS, dev)
    idx = torch.empty((T, top_k), dtype=torch.int32, device=dev)
    w = torch.empty((T, top_k), dtype=torch.float32, device=dev)
    n = torch.empty(E, dtype=torch.int32, device=dev) if counts else None
    a = _native.SelectArgs(_ptr(logits), _ptr(bias), _ptr(idx), _ptr(w), _ptr(n), _ld(logits), T, E, top_k,
                           _type(logits), _type(bias), _SCORES[score], n_group, topk_group,
                           _GROUP_SCORES[group_score], bool(renormalize), scale)
    _done(_native.lib().moe_b200_select_experts(ctypes.byref(a), _stream(dev)), "select_experts")
    return Selection(idx, w, n)


@torch.no_grad()
def select_experts_backward(dw: torch.Tensor, logits: torch.Tensor, idx: torch.Tensor, *, score: str = "sigmoid",
                            renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """The gradient of :func:`select_experts`' weights with respect to the logits, from ``dw``
    (float32 [T, top_k]) and the ids it chose.  The choice itself has no gradient."""
    _rows(logits, "logits")
    T, E = logits.shape
    dev = logits.device
    _check(score in _SCORES, "score must be 'sigmoid' or 'softmax'")
    _check(idx.dim() == 2 and idx.shape[0] == T and idx.dtype == torch.int32 and idx.is_contiguous()
           and idx.device == dev, "idx must be a contiguous int32 [T, top_k] tensor on the device")
    _check(dw.shape == idx.shape and dw.dtype == torch.float32 and dw.is_contiguous() and dw.device == dev,
           "dw must be a contiguous float32 [T, top_k] tensor on the device")
    out = torch.empty((T, E), dtype=logits.dtype, device=dev)
    a = _native.SelectBackwardArgs(_ptr(logits), _ptr(idx), _ptr(dw), _ptr(out), _ld(logits), E, T, E, idx.shape[1],
                                   _type(logits), _SCORES[score], bool(renormalize), scale)
    _done(_native.lib().moe_b200_select_experts_backward(ctypes.byref(a), _stream(dev)), "select_experts_backward")
    return out


@torch.no_grad()
def quantize_int8(x: torch.Tensor, *, swiglu: bool = False):
    """8-bit codes and scales of the rows of ``x``: (int8 [rows, cols], float32 [rows]) with
    scale = max(amax / 127, 2**-126).  With ``swiglu``, of silu(x[:, cols:]) * x[:, :cols] (the
    expert layer's order of the two halves).  For weights [out, in] the rows are the channels."""
    _rows(x, "x")
    dev = x.device
    rows, cols = x.shape
    if swiglu:
        _check(cols % 2 == 0, "swiglu needs an even number of columns")
        cols //= 2
    q = torch.empty((rows, cols), dtype=torch.int8, device=dev)
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    a = _native.QuantizeArgs(_ptr(x), _ptr(q), _ptr(scale), _ld(x), cols, rows, cols, _type(x), bool(swiglu))
    _done(_native.lib().moe_b200_quantize_int8(ctypes.byref(a), _stream(dev)), "quantize_int8")
    return q, scale


@torch.no_grad()
def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                x_scale: torch.Tensor | None = None, bias: torch.Tensor | None = None, swiglu: bool = False,
                out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t, n] = x_scale[t] * weight_scale[n] * sum_k q[t, k] * weight[n, k] + bias[n]``.

    ``weight`` is int8 [N, K] with ``weight_scale`` float32 [N].  ``x`` is int8 [T, K] with
    ``x_scale`` float32 [T], or bf16 / fp16 / fp32 and quantised per token in the call
    (:func:`quantize_int8`; [T, 2 K] with ``swiglu``).  The integer sums are exact.  K must be a
    multiple of 16 and rows of int8 tensors start on 16-byte boundaries.  ``out_dtype``: bf16 by
    default (x's type if that is fp16 or fp32).
    """
    _rows(x, "x", dtypes=(*_FLOATS, torch.int8))
    dev = x.device
    _rows(weight, "weight", dtypes=(torch.int8,), dev=dev)
    T, N, K = x.shape[0], weight.shape[0], weight.shape[1]
    _check(x.shape[1] == (2 * K if swiglu else K), "x and weight do not fit")
    _vector(weight_scale, "weight_scale", N, (torch.float32,), dev)
    _check(weight_scale is not None, "weight_scale is required")
    if x.dtype == torch.int8:
        _check(x_scale is not None, "an int8 x needs x_scale")
        _vector(x_scale, "x_scale", T, (torch.float32,), dev)
    else:
        _check(x_scale is None, "x_scale is computed for a floating-point x")
    _vector(bias, "bias", N, _FLOATS, dev)
    if out is None:
        if out_dtype is None:
            out_dtype = torch.bfloat16 if x.dtype == torch.int8 else x.dtype
        _check(out_dtype in _FLOATS, f"unsupported out_dtype {out_dtype}")
        out = torch.empty((T, N), dtype=out_dtype, device=dev)
    else:
        _result(out, "out", (T, N), _FLOATS if out_dtype is None else (out_dtype,), dev)
    if T == 0 or N == 0:
        return out
    lib = _native.lib()
    n = lib.moe_b200_int8_linear_workspace_size(T, N, K, _type(x))
    _check(n > 0, "unsupported sizes")
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    a = _native.LinearArgs(_ptr(x), _ptr(x_scale), _ptr(weight), _ptr(weight_scale), _ptr(bias), _ptr(out), _ld(x),
                           _ld(weight), _ld(out), T, N, K, _type(x), _type(out), _type(bias), bool(swiglu))
    _done(lib.moe_b200_int8_linear(ctypes.byref(a), ws.data_ptr(), ws.numel(), _stream(dev)), "int8_linear")
    return out


def operator_status(device=None, clear: bool = True) -> int:
    """Synchronises and returns the status word of this module's operators on the device: 0, or
    the code of a bounded device-side wait that gave up (the call's result is then not valid)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        rc = int(_native.lib().moe_b200_operator_status(_stream(dev), 1 if clear else 0))
    if rc < 0:
        raise RuntimeError(f"operator_status failed ({-rc}): {_native.last_error()}")
    return rc
