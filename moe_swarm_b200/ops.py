"""Operators that stand around the expert layer in a transformer block: the norms with the
block's gate and residual sum, the choice of experts, and linear layers in 8-bit integers.

Like ``run``, they check their arguments (:class:`MoEArgumentError`), run on the current CUDA
stream without a host synchronisation, and compute in the hand-written CUDA of
``libmoe_b200.so``; there is no CPU or PyTorch path.  Tensors are ``[rows, cols]`` with adjacent
elements in a row; rows may be further apart than their length (slices of wider tensors).
The backward functions are explicit: they take what the forward took and the gradients of its
results.  Nothing here records a graph, so a tensor that requires a gradient is refused while gradients are
enabled (call under ``torch.no_grad()``, or inside a ``torch.autograd.Function``); the backward functions
refuse incoming gradients that do.
"""

from __future__ import annotations

import functools
import threading
from typing import NamedTuple

import torch

from . import _native

_TYPES = {torch.bfloat16: _native.BF16, torch.float16: _native.FP16, torch.float32: _native.FP32,
          torch.float8_e4m3fn: _native.E4M3, torch.int8: _native.INT8}
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_FP32, _INT8, _LINEAR_IN = (torch.float32,), (torch.int8,), (*_FLOATS, torch.int8)


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


# The checks run on every call, and a decode step's kernels take a few microseconds: each is one
# expression, messages are put together only on refusal, devices are compared by index.

def _rows(t, name: str, shape=None, dtypes=_FLOATS, dev=None):
    """Checks a [rows, cols] CUDA tensor of the call; returns its row pitch in elements (which
    says nothing for a single row)."""
    st = t.stride()
    if (len(st) != 2 or (st[1] != 1 and t.shape[1] > 1) or t.dtype not in dtypes
            or (not t.is_cuda if dev is None else t.get_device() != dev)
            or (shape is not None and t.shape != shape)):
        _check(len(st) == 2 and (st[1] == 1 or t.shape[1] < 2),
               f"{name} must be [rows, cols] with adjacent elements in a row")
        _check(shape is None or t.shape == shape, f"{name} must be {list(shape or ())}")
        _check(t.dtype in dtypes, f"{name} has an unsupported type {t.dtype}")
        _check(t.is_cuda, "all tensors must be CUDA tensors (there is no CPU path)")
        raise MoEArgumentError("all tensors must be on one device")
    return st[0]


def _like(t, dtype=None):
    """A new tensor of t's shape without gaps.  (empty_like would order the strides of rows that overlap,
    such as a sliding window's, as it finds them: by columns.)"""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else t.new_empty(t.shape, dtype=dtype)


def _no_graph(what: str, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise MoEArgumentError(f"{what} records no graph, and a tensor of the call requires a gradient: call it "
                                       "under torch.no_grad() and its backward function explicitly")


def _result(t, name: str, shape, dtypes, dev):
    """Checks a tensor that receives a result: rows may not overlap.  Returns its row pitch."""
    ld = _rows(t, name, shape, dtypes, dev)
    if shape[0] > 1 and ld < shape[1]:
        raise MoEArgumentError(f"{name}: rows overlap")
    return ld


def _vector(t, name: str, n: int, dtypes, dev):
    if t is None:
        raise MoEArgumentError(f"{name} is required")
    if t.shape != (n,) or (n > 1 and t.stride(0) != 1) or t.dtype not in dtypes or t.get_device() != dev:
        _check(t.dim() == 1 and t.shape[0] == n and t.is_contiguous(), f"{name} must be a contiguous [{n}] tensor")
        _check(t.dtype in dtypes, f"{name} has an unsupported type {t.dtype}")
        raise MoEArgumentError("all tensors must be on one device")


def _matrix(t, name: str, shape, dtype, dev):
    """Checks a contiguous matrix (the tensors that the layer's routing results are made of)."""
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.get_device() != dev:
        raise MoEArgumentError(f"{name} must be a contiguous {dtype} {list(shape)} tensor on the device")


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _type(t) -> int:
    return 0 if t is None else _TYPES[t.dtype]


_functions: dict = {}   # operator -> its C entry, looked up once


def _call(fn: str, dev: int, args, *workspace):
    """Calls moe_b200_<fn> on the device's current stream, with that device current."""
    f = _functions.get(fn)
    if f is None:
        f = _functions[fn] = _native.packed_entry(fn, bool(workspace))
    if torch._C._cuda_getDevice() == dev:
        rc = f(args, *workspace, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = f(args, *workspace, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        raise _failure(rc, fn)


@functools.lru_cache(maxsize=256)
def _workspace_size(fn: str, *sizes: int) -> int:
    return getattr(_native.lib(), f"moe_b200_{fn}_workspace_size")(*sizes)


_SCRATCH_KEPT = 4 << 20   # bytes kept per (device, stream, thread)
_scratch: dict[tuple[int, int, int], torch.Tensor] = {}


def _workspace(n: int, dev: int) -> torch.Tensor:
    """Scratch of n bytes for a call on the device's current stream.  Small ones are kept per
    (device, stream, host thread): such calls are enqueued, and run, one after another, while two
    threads could enqueue the kernels of their calls in turn.  Large ones, and those of a graph
    capture (whose replays would share them with later calls), are allocated per call; so are those of
    another device than the current one, the one whose stream can be asked whether it captures."""
    if n > _SCRATCH_KEPT or torch._C._cuda_getDevice() != dev or torch._C._cuda_isCurrentStreamCapturing():
        return torch.empty(n, dtype=torch.uint8, device=dev)
    key = (dev, torch._C._cuda_getCurrentRawStream(dev), threading.get_ident())
    ws = _scratch.get(key)
    if ws is None:
        ws = _scratch[key] = torch.empty(_SCRATCH_KEPT, dtype=torch.uint8, device=dev)
    return ws


def _failure(rc: int, what: str) -> Exception:
    if rc == _native.ERR_ARG:
        return MoEArgumentError(f"{what}: {_native.last_error()}")
    return RuntimeError(f"{what} failed ({rc}): {_native.last_error()}")


def _gate_layout(gate, rows: int, cols: int, dev: int):
    """(row stride, varies along a row) of a gate [cols], [1, cols], [rows, 1], [1, 1] or [rows, cols]."""
    _check(gate.dtype in _FLOATS, "gate has an unsupported type")
    _check(gate.get_device() == dev, "all tensors must be on one device")
    size, st = gate.shape, gate.stride()
    if len(st) == 1:
        size, st = (1, *size), (0, *st)
    _check(len(st) == 2 and size[0] in (1, rows) and size[1] in (1, cols),
           "gate must be broadcastable to [rows, cols]")
    per_column = cols > 1 and size[1] == cols
    per_row = rows > 1 and size[0] == rows
    _check(not per_column or st[1] == 1, "gate must have adjacent elements in a row")
    _check(not per_row or st[0] > 0, "gate: pass a broadcast gate with its own size, not expanded")
    return st[0] if per_row else 0, int(per_column)


def block_norm(y: torch.Tensor | None, residual: torch.Tensor | None, *, post_weight: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, scale: float = 1.0, pre_weight: torch.Tensor | None = None,
               eps: float = 1e-6, weight_offset: float = 0.0, x_dtype: torch.dtype | None = None,
               residual_out: torch.Tensor | None = None, out: torch.Tensor | None = None) -> BlockNormOut:
    """The end of one block and the beginning of the next, in one pass::

        n  = rms_norm(y) * (post_weight + weight_offset)      (n = y without post_weight)
        r' = residual + scale * gate * n
        x  = rms_norm(r') * (pre_weight + weight_offset)      (no x without pre_weight)

    ``y`` [rows, cols] is the block's output (None: x is the norm of ``residual``), ``residual``
    may have another type (None: 0; fp32 if y is), ``gate`` is [cols], [1, cols], [rows, 1], [1, 1] or [rows, cols].
    ``x_dtype`` is the type of x (y's by default); ``torch.float8_e4m3fn`` quantises x per row and
    128 columns and returns ``x_scale`` [ceil(cols / 128), rows]: the ``hidden_states`` and
    ``hidden_states_scale`` of :func:`moe_swarm_b200.run`.  ``residual_out`` (may be ``residual``)
    and ``out`` receive r' and x instead of new tensors.
    """
    _no_graph("block_norm", y, residual, post_weight, gate, pre_weight, residual_out, out)
    first = residual if y is None else y
    _check(first is not None, "y or residual is required")
    shape, dev = first.shape, first.get_device()
    y_ld = r_ld = ro_ld = x_ld = 0
    if y is not None:
        y_ld = _rows(y, "y")
        if residual is not None:
            r_ld = _rows(residual, "residual", shape, _FP32 if y.dtype == torch.float32 else _FLOATS, dev)
    else:
        r_ld = _rows(residual, "residual")
    rows, cols = shape
    if post_weight is not None:
        _vector(post_weight, "post_weight", cols, _FLOATS, dev)
    gate_ld, gate_cols = (0, 0) if gate is None else _gate_layout(gate, rows, cols, dev)
    stream = y if residual is None else residual   # the tensor that r' is like
    if y is None:
        _check(residual_out is None, "residual_out is the residual itself without y")
    elif residual_out is None:
        residual_out, ro_ld = _like(stream), cols
    else:
        ro_ld = _result(residual_out, "residual_out", shape, (stream.dtype,), dev)
    x = x_scale = None
    if pre_weight is not None:
        _vector(pre_weight, "pre_weight", cols, _FLOATS, dev)
        if x_dtype is None:
            x_dtype = first.dtype if out is None else out.dtype
        _check(x_dtype in _TYPES and x_dtype != torch.int8, "unsupported x_dtype")
        if out is None:
            x, x_ld = _like(first, x_dtype), cols
        else:
            x, x_ld = out, _result(out, "out", shape, (x_dtype,), dev)
        if x_dtype == torch.float8_e4m3fn:
            x_scale = first.new_empty(((cols + 127) // 128, rows), dtype=torch.float32)
    _call("block_norm", dev, _native.NormArgs.pack(
        _ptr(y), _ptr(residual), _ptr(post_weight), _ptr(pre_weight), _ptr(gate), _ptr(residual_out), _ptr(x),
        _ptr(x_scale), y_ld, r_ld, ro_ld, x_ld, gate_ld, rows, cols, _TYPES[first.dtype], _TYPES[stream.dtype],
        _type(post_weight), _type(pre_weight), _type(gate), _type(x), gate_cols, scale, eps, weight_offset))
    return BlockNormOut(residual if y is None else residual_out, x, x_scale)


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
    _no_graph("block_norm_backward", dx, dresidual)
    r_ld = _rows(residual, "residual")
    shape, dev, r_dtype = residual.shape, residual.get_device(), residual.dtype
    rows, cols = shape
    y_dtype = (residual if y is None and dx is None else dx if y is None else y).dtype
    _check(r_dtype is torch.float32 or y_dtype is not torch.float32, "with a y of fp32 the residual must be fp32")
    _check(dx is not None or dresidual is not None, "dx or dresidual is required")
    _check(dx is None or pre_weight is not None, "dx needs pre_weight")
    _check(y is not None or (post_weight is None and gate is None), "post_weight and gate need y")
    y_ld = 0 if y is None else _rows(y, "y", shape, (y_dtype,), dev)
    dx_ld = 0 if dx is None else _rows(dx, "dx", shape, (y_dtype,), dev)
    dr_ld = 0 if dresidual is None else _rows(dresidual, "dresidual", shape, (r_dtype,), dev)
    dy = dpre = dpost = dgate = None
    gate_ld = gate_cols = 0
    dres = _like(residual)
    if y is not None:
        dy = _like(y)
    if dx is not None:
        _vector(pre_weight, "pre_weight", cols, _FLOATS, dev)
        dpre = torch.empty_like(pre_weight, dtype=torch.float32)
    if post_weight is not None:
        _vector(post_weight, "post_weight", cols, _FLOATS, dev)
        dpost = torch.empty_like(post_weight, dtype=torch.float32)
    if gate is not None:
        gate_ld, gate_cols = _gate_layout(gate, rows, cols, dev)
        dgate = gate.new_empty(gate.shape, dtype=gate.dtype if gate_ld and gate_cols else torch.float32)
    n = _workspace_size("block_norm_backward", rows, cols)
    _check(n > 0, "unsupported sizes")
    ws = _workspace(n, dev)
    _call("block_norm_backward", dev, _native.NormBackwardArgs.pack(
        _ptr(dx), _ptr(dresidual), _ptr(residual), _ptr(y), _ptr(post_weight), _ptr(pre_weight), _ptr(gate),
        _ptr(dres), _ptr(dy), _ptr(dpre), _ptr(dpost), _ptr(dgate), dx_ld, dr_ld, r_ld, y_ld, gate_ld, cols, cols,
        cols, rows, cols, _TYPES[y_dtype], _TYPES[r_dtype], _type(post_weight), _type(pre_weight), _type(gate),
        gate_cols, scale, eps, weight_offset), ws.data_ptr(), ws.numel())
    return BlockNormGrads(dres, dy, dpre, dpost, dgate)


_SCORES = {"sigmoid": 0, "softmax": 1}
_GROUP_SCORES = {"top2": 0, "max": 1}


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
    _no_graph("select_experts", logits, bias)
    ld = _rows(logits, "logits")
    T, E = logits.shape
    dev = logits.get_device()
    _check(score in _SCORES, "score must be 'sigmoid' or 'softmax'")
    _check(group_score in _GROUP_SCORES, "group_score must be 'top2' or 'max'")
    _check(1 <= top_k <= E, "top_k must be in [1, number of experts]")
    _check(1 <= topk_group <= n_group <= E, "topk_group must be in [1, n_group], n_group in [1, number of experts]")
    if bias is not None:
        _vector(bias, "bias", E, _FLOATS, dev)
    idx = logits.new_empty((T, top_k), dtype=torch.int32)
    w = logits.new_empty((T, top_k)) if logits.dtype == torch.float32 else torch.empty_like(idx, dtype=torch.float32)
    n = idx.new_empty(E) if counts else None
    _call("select_experts", dev, _native.SelectArgs.pack(
        logits.data_ptr(), _ptr(bias), idx.data_ptr(), w.data_ptr(), _ptr(n), ld, T, E, top_k, _TYPES[logits.dtype],
        _type(bias), _SCORES[score], n_group, topk_group, _GROUP_SCORES[group_score], bool(renormalize), scale))
    return Selection(idx, w, n)


def select_experts_backward(dw: torch.Tensor, logits: torch.Tensor, idx: torch.Tensor, *, score: str = "sigmoid",
                            renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """The gradient of :func:`select_experts`' weights with respect to the logits, from ``dw``
    (float32 [T, top_k]) and the ids it chose.  The choice itself has no gradient."""
    _no_graph("select_experts_backward", dw)
    ld = _rows(logits, "logits")
    T, E = logits.shape
    dev = logits.get_device()
    _check(score in _SCORES, "score must be 'sigmoid' or 'softmax'")
    _check(idx.dim() == 2, "idx must be [T, top_k]")
    _matrix(idx, "idx", (T, idx.shape[1]), torch.int32, dev)
    _matrix(dw, "dw", idx.shape, torch.float32, dev)
    out = _like(logits)
    _call("select_experts_backward", dev, _native.SelectBackwardArgs.pack(
        logits.data_ptr(), idx.data_ptr(), dw.data_ptr(), out.data_ptr(), ld, E, T, E, idx.shape[1],
        _TYPES[logits.dtype], _SCORES[score], bool(renormalize), scale))
    return out


def quantize_int8(x: torch.Tensor, *, swiglu: bool = False):
    """8-bit codes and scales of the rows of ``x``: (int8 [rows, cols], float32 [rows]) with
    scale = max(amax / 127, 2**-126).  With ``swiglu``, of silu(x[:, cols:]) * x[:, :cols] (the
    expert layer's order of the two halves).  For weights [out, in] the rows are the channels.
    Without ``swiglu`` the codes are those of 64-bit arithmetic with amax * (1 / 127) for a scale."""
    _no_graph("quantize_int8", x)
    ld = _rows(x, "x")
    dev = x.get_device()
    rows, cols = x.shape
    if swiglu:
        _check(cols % 2 == 0, "swiglu needs an even number of columns")
        cols //= 2
    q = x.new_empty((rows, cols), dtype=torch.int8)
    scale = x.new_empty(rows, dtype=torch.float32)
    _call("quantize_int8", dev, _native.QuantizeArgs.pack(x.data_ptr(), q.data_ptr(), scale.data_ptr(), ld, cols, rows, cols,
                                                     _TYPES[x.dtype], bool(swiglu)))
    return q, scale


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
    _no_graph("int8_linear", x, weight_scale, x_scale, bias, out)
    x_ld = _rows(x, "x", None, _LINEAR_IN)
    dev = x.get_device()
    w_ld = _rows(weight, "weight", None, _INT8, dev)
    T, (N, K) = x.shape[0], weight.shape
    _check(x.shape[1] == (2 * K if swiglu else K), "x and weight do not fit")
    _vector(weight_scale, "weight_scale", N, _FP32, dev)
    x_type = _TYPES[x.dtype]
    if x_type == _native.INT8:
        _check(x_scale is not None, "an int8 x needs x_scale")
        _vector(x_scale, "x_scale", T, _FP32, dev)
    else:
        _check(x_scale is None, "x_scale is computed for a floating-point x")
    if bias is not None:
        _vector(bias, "bias", N, _FLOATS, dev)
    if out is None:
        if out_dtype is None:
            out_dtype = torch.bfloat16 if x_type == _native.INT8 else x.dtype
        _check(out_dtype in _FLOATS, "unsupported out_dtype")
        out, out_ld = x.new_empty((T, N)) if out_dtype == x.dtype else x.new_empty((T, N), dtype=out_dtype), N
    else:
        out_ld = _result(out, "out", (T, N), _FLOATS if out_dtype is None else (out_dtype,), dev)
    if T == 0 or N == 0:
        return out
    n = _workspace_size("int8_linear", T, N, K, x_type)
    _check(n > 0, "unsupported sizes")
    ws = _workspace(n, dev)
    _call("int8_linear", dev, _native.LinearArgs.pack(
        x.data_ptr(), _ptr(x_scale), weight.data_ptr(), weight_scale.data_ptr(), _ptr(bias), out.data_ptr(), x_ld, w_ld,
        out_ld, T, N, K, x_type, _TYPES[out.dtype], _type(bias), bool(swiglu)), ws.data_ptr(), ws.numel())
    return out


def operator_status(device=None, clear: bool = True) -> int:
    """Synchronises and returns the status word of this module's operators on the device: 0, or
    the code of a bounded device-side wait that gave up (the call's result is then not valid)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        rc = int(_native.lib().moe_b200_operator_status(stream, 1 if clear else 0))
    if rc < 0:
        raise RuntimeError(f"operator_status failed ({-rc}): {_native.last_error()}")
    return rc
