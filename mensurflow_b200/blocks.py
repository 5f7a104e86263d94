"""Operators of language models, on B200 tensors: the gated feed-forward block with its backward
pass, the orthogonalised update and the embedding with its gradient, beside ``linear`` and
``linear_backward``.

They follow the package's manner: fp32 CUDA tensors, work queued on the current stream of the
tensors' device, explicit backward functions, ``ValueError`` for bad arguments and
``NotImplementedError`` where there is no kernel. Views with a unit stride in either of a matrix's
two dimensions (row-major, transposed, sliced) go to the kernels as they are; others are packed
first. The reference has no counterpart of these operators (it composes blocks from gemm and
elementwise calls).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import GatedFfnDesc, GatedFfnGrads, check
from .ops import _kernel_for, _require, _same, contiguous

_GATED_ACTS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "relu": _lib.ACT_RELU,
               "gelu": _lib.ACT_GELU, "gelu_tanh": _lib.ACT_GELU_TANH, "silu": _lib.ACT_SILU}


def _run(device: torch.device, op: str, call, *args) -> None:
    """call(*args, stream) with the current stream of `device`, which is made current first. These
    operators run for a few microseconds at their smallest, so the usual case costs no context
    manager and no Stream object."""
    if torch.cuda.current_device() == device.index:
        status = call(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            status = call(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if status:
        check(status, op)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return t.data_ptr() if t is not None and t.numel() else None


def _lies(t: torch.Tensor) -> Optional[bool]:
    """False: rows are contiguous, True: columns are, None: neither."""
    if t.stride(1) == 1 or t.shape[1] <= 1:
        return False
    return True if t.stride(0) == 1 or t.shape[0] <= 1 else None


def _unit(t: torch.Tensor) -> torch.Tensor:
    """t itself when one of its strides is 1, else a packed copy."""
    return contiguous(t) if _lies(t) is None else t


def _strides(t: torch.Tensor):
    """Strides for the kernels: a dimension of one entry has none that matters."""
    rows, cols = t.shape
    cs = 1 if cols <= 1 else t.stride(1)
    rs = max(cols, 1) if rows <= 1 and cs == 1 else t.stride(0)
    return rs, cs


class GatedSaved:
    """What ``gated_ffn(..., save=True)`` keeps for the backward pass: the gate's and the up
    projection's results, in the kernels' own order, in a device tensor (``buffer``)."""

    def __init__(self, buffer: torch.Tensor, rows: int, features: int, activation):
        self.buffer = buffer
        self.rows = rows
        self.features = features
        self.activation = activation


def _gated_fast(x, w_gate, w_up, w_down, activation, transpose_w):
    """The descriptor of a call whose tensors are all contiguous fp32 matrices of one device that
    fit each other; None for any other call, which `_gated_args` checks and lays out."""
    try:
        rows, d = x.shape
        f = w_gate.shape[0 if transpose_w else 1]
        inner, outer = ((f, d), (d, f)) if transpose_w else ((d, f), (f, d))
        if not (x.is_cuda and rows > 0 and d > 1 and f > 1 and w_gate.shape == inner and
                w_up.shape == inner and w_down.shape == outer):
            return None
        device = x.device
        for t in (x, w_gate, w_up, w_down):
            if t.dtype is not torch.float32 or not t.is_contiguous() or t.device != device:
                return None
        ws, ds = ((1, d), (1, f)) if transpose_w else ((f, 1), (d, 1))
        return GatedFfnDesc(x.data_ptr(), d, 1, w_gate.data_ptr(), *ws, w_up.data_ptr(), *ws,
                            w_down.data_ptr(), *ds, rows, d, f, _GATED_ACTS[activation], 0)
    except (AttributeError, IndexError, KeyError, TypeError, ValueError):
        return None


def _gated_args(op, x, w_gate, w_up, w_down, activation, transpose_w):
    desc = _gated_fast(x, w_gate, w_up, w_down, activation, transpose_w)
    if desc is not None:
        return desc, (x, w_gate, w_up, w_down)
    _require(x, op, "x", 1, at_least=True)
    for t, name in ((w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")):
        _require(t, op, name, 2)
    _same(op, x, w_gate, w_up, w_down)
    if activation not in _GATED_ACTS:
        raise ValueError(f"{op}: unknown activation {activation!r}")
    gate, up, down = (t.t() if transpose_w else t for t in (w_gate, w_up, w_down))
    d, f = gate.shape
    if x.shape[-1] != d:
        raise ValueError(f"{op}: x {tuple(x.shape)} does not fit w_gate {tuple(w_gate.shape)}")
    if tuple(up.shape) != (d, f):
        raise ValueError(f"{op}: w_up {tuple(w_up.shape)} differs from w_gate "
                         f"{tuple(w_gate.shape)}")
    if tuple(down.shape) != (f, d):
        raise ValueError(f"{op}: w_down {tuple(w_down.shape)} does not fit w_gate "
                         f"{tuple(w_gate.shape)}")
    _kernel_for(op, x)
    rows = 1
    for s in x.shape[:-1]:
        rows *= s
    x2 = _rows_of(x, rows, d)
    if _lies(x2):  # a scale for every row: rows have to be contiguous
        x2 = contiguous(x2)
    gate, up, down = _unit(gate), _unit(up), _unit(down)
    if _lies(gate) != _lies(up):  # the two projections share a tile: one way round
        gate, up = contiguous(gate), contiguous(up)
    desc = GatedFfnDesc()
    desc.x = _ptr(x2)
    desc.x_rs, desc.x_cs = _strides(x2)
    desc.w_gate, desc.w_up, desc.w_down = _ptr(gate), _ptr(up), _ptr(down)
    desc.w_gate_rs, desc.w_gate_cs = _strides(gate)
    desc.w_up_rs, desc.w_up_cs = _strides(up)
    desc.w_down_rs, desc.w_down_cs = _strides(down)
    desc.rows, desc.d, desc.f = rows, d, f
    desc.activation = _GATED_ACTS[activation]
    return desc, (x2, gate, up, down)


def _rows_of(t: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """t [..., cols] as a matrix [rows, cols] with a unit stride: a view where there is one."""
    if t.dim() == 2:
        return _unit(t)
    if t.numel() and not t.is_contiguous():
        try:
            return _unit(t.view(rows, cols))
        except RuntimeError:
            t = contiguous(t)
    return t.reshape(rows, cols)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: Optional[str] = "silu", *, transpose_w: bool = False,
              save: bool = False):
    """(act(x @ w_gate) * (x @ w_up)) @ w_down: the gated feed-forward block. x is [..., d],
    w_gate and w_up are [d, f], w_down is [f, d]; with ``transpose_w`` the weights are stored
    [outputs, inputs], as in ``linear``. ``activation``: "silu", "gelu" (exact), "gelu_tanh",
    "relu" or None. Both projections, the activation and their product are one kernel; its result
    never leaves the split form the down projection reads.

    With ``save`` the result is (y, saved): ``saved`` spares ``gated_ffn_backward`` the two
    projections at the price of 8 bytes per row and feature.

    The products are fp32-faithful (fp16 pairs under power-of-two scales, sums in fp32), whatever
    ``set_default_precision`` says. Rows of x and of the hidden values have scales of their own, so
    no row of the result depends on another; a weight more than 2^17 below the largest of its
    128 x 128 block keeps an absolute error of 2^-39 of that one. Non-finite inputs give non-finite
    results, though an infinity may come out as NaN. Up to 16 rows, without ``save``, run as plain
    fp32 sums at the speed the weights are read."""
    desc, keep = _gated_args("gated_ffn", x, w_gate, w_up, w_down, activation, transpose_w)
    rows, d, f = desc.rows, desc.d, desc.f
    so = _lib.lib()
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    saved = None
    if save:
        saved = GatedSaved(x.new_empty(so.mfk_gated_ffn_saved_floats(rows, f)), rows, f, activation)
    _run(x.device, "gated_ffn", so.mfk_gated_ffn_f32, ctypes.byref(desc), _ptr(y), d or 1,
         _ptr(saved.buffer) if save else None)
    return (y, saved) if save else y


def gated_ffn_backward(grad: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor,
                       w_up: torch.Tensor, w_down: torch.Tensor,
                       activation: Optional[str] = "silu", *, saved: Optional[GatedSaved] = None,
                       transpose_w: bool = False, need_x: bool = True, need_w: bool = True):
    """(dx, dw_gate, dw_up, dw_down) of ``gated_ffn`` for grad = dL/dy, with the forward call's
    arguments; dx has x's shape and the weights' gradients have the weights' own layouts.
    ``saved`` from the forward call with the same x and weights; without it the two projections
    are computed again. What is not needed is None. A row whose gradient is all zero (padding) adds
    nothing to the weights' gradients, whatever x holds there, and its dx is zero. Arithmetic as in
    ``gated_ffn``, with one scale per 128 x 128 block: an entry of grad more than 2^17 below the
    largest of its block keeps an absolute error of 2^-39 of that one, an entry of the hidden values
    and their gradients more than 2^14 below one of 2^-36."""
    op = "gated_ffn_backward"
    desc, keep = _gated_args(op, x, w_gate, w_up, w_down, activation, transpose_w)
    _require(grad, op, "grad")
    _same(op, x, grad)
    if tuple(grad.shape) != tuple(x.shape):
        raise ValueError(f"{op}: grad {tuple(grad.shape)} differs from x {tuple(x.shape)}")
    rows, d, f = desc.rows, desc.d, desc.f
    if saved is not None:
        if not isinstance(saved, GatedSaved):
            raise TypeError(f"{op}: saved must come from gated_ffn(..., save=True)")
        if (saved.rows, saved.features) != (rows, f) or saved.buffer.device != x.device or \
                saved.buffer.dtype is not torch.float32 or not saved.buffer.is_contiguous() or \
                saved.buffer.numel() != _lib.lib().mfk_gated_ffn_saved_floats(rows, f) or \
                _GATED_ACTS[saved.activation] != desc.activation:
            raise ValueError(f"{op}: saved belongs to another call ({saved.rows} rows, "
                             f"{saved.features} features, {saved.activation})")
    if not need_x and not need_w:
        return None, None, None, None
    g2 = _rows_of(grad, rows, d)
    o = GatedFfnGrads()
    o.grad = _ptr(g2)
    o.grad_rs, o.grad_cs = _strides(g2)
    dx = dw_gate = dw_up = dw_down = None
    if need_x:
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        o.dx, o.ld_dx = _ptr(dx), max(d, 1)
    if need_w:
        dw_gate, dw_up, dw_down = (torch.empty_like(t, memory_format=torch.contiguous_format)
                                   for t in (w_gate, w_up, w_down))
        o.dw_gate, o.dw_up, o.dw_down = _ptr(dw_gate), _ptr(dw_up), _ptr(dw_down)
        o.dw_rs, o.dw_cs = (1, max(d, 1)) if transpose_w else (max(f, 1), 1)
        o.dw_down_rs, o.dw_down_cs = (1, max(f, 1)) if transpose_w else (max(d, 1), 1)
    _run(x.device, op, _lib.lib().mfk_gated_ffn_backward_f32, ctypes.byref(desc),
         ctypes.byref(o), _ptr(saved.buffer) if saved else None)
    return dx, dw_gate, dw_up, dw_down


def orthogonalize(update: torch.Tensor, steps: int = 5,
                  coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7) -> torch.Tensor:
    """The update with its singular values drawn towards 1 by Newton-Schulz products: for each
    matrix of ``update`` [..., m, n], x = u / (||u||_F + eps), then ``steps`` times
    x <- a x + (b g + c g g) x with g = x x^T and (a, b, c) = ``coefficients`` (on the transpose
    where m > n). All matrices of a batch run in the same launches. The Gram matrix and its square
    are symmetric: only their lower halves are computed. Arithmetic as in ``gated_ffn``."""
    op = "orthogonalize"
    _require(update, op, "update", 2, at_least=True)
    if not isinstance(steps, int) or isinstance(steps, bool) or not 1 <= steps < 2 ** 31:
        raise ValueError(f"{op}: steps must be a whole number of at least 1 and below 2^31, "
                         f"got {steps!r}")
    if len(coefficients) != 3:
        raise ValueError(f"{op}: coefficients must be (a, b, c)")
    if not eps >= 0:
        raise ValueError(f"{op}: eps must be at least 0, got {eps!r}")
    _kernel_for(op, update)
    m, n = update.shape[-2:]
    if update.numel() == 0:
        return torch.empty_like(update, memory_format=torch.contiguous_format)
    if n > 1 and update.stride(-1) != 1 and (update.stride(-2) == 1 or m <= 1):
        return orthogonalize(update.transpose(-2, -1), steps, coefficients,
                             eps).transpose(-2, -1)
    u = update
    if n > 1 and u.stride(-1) != 1:
        u = contiguous(u)
    try:
        u = u.view(-1, m, n)
    except RuntimeError:
        u = contiguous(u).view(-1, m, n)
    out = torch.empty_like(update, memory_format=torch.contiguous_format)
    batch = u.shape[0]
    a, b, c = (float(v) for v in coefficients)
    _run(update.device, op, _lib.lib().mfk_orthogonalize_f32, u.data_ptr(), batch, m, n,
         u.stride(1) if m > 1 else n, u.stride(0) if batch > 1 else 0, out.data_ptr(), n, m * n,
         steps, a, b, c, float(eps))
    return out


def _ids(op: str, ids: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    _require(ids, op, "ids")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{op}: ids must be int64 or int32, got {ids.dtype}")
    if ids.device != like.device:
        raise ValueError(f"{op}: tensors are on different devices; move one with Tensor::to()")
    return ids.contiguous()


def embedding(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * table[ids]: the rows of ``table`` [rows, d] that ``ids`` (any shape, int64 or int32)
    names, [*ids.shape, d]. An id outside the table gives a row of zeros and sets the bit
    ``MFK_DEVERR_INDEX`` of ``device_status()``."""
    op = "embedding"
    try:  # the usual call, checked in one go
        plain = (table.dtype is torch.float32 and table.is_cuda and table.dim() == 2 and
                 ids.dtype in (torch.int64, torch.int32) and ids.device == table.device and
                 ids.is_contiguous())
    except AttributeError:
        plain = False
    if plain:
        index = ids
    else:
        _require(table, op, "table", 2)
        index = _ids(op, ids, table)
        _kernel_for(op, table)
    rows, d = table.shape
    n = index.numel()
    if rows == 0 and n and d:
        raise ValueError(f"{op}: the table has no rows")
    t = table if d <= 1 or table.stride(1) == 1 else contiguous(table)
    out = table.new_empty(ids.shape + (d,))
    if n and d:
        _run(table.device, op, _lib.lib().mfk_embedding_f32, t.data_ptr(), rows, d,
             t.stride(0) if rows > 1 else d, index.data_ptr(), index.element_size(), n,
             float(scale), out.data_ptr(), d)
    return out


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0, *,
                   padding: Optional[int] = None) -> torch.Tensor:
    """The gradient of ``embedding``'s table, [rows, d]: scale times the sum of ``grad``
    [*ids.shape, d] over the tokens of each id, zeros for ids that do not occur. Tokens of the id
    ``padding`` take no part. Sums are fp32 over tokens sorted by id, in an order fixed by the ids:
    repeated calls give the same bits. An id outside the table takes no part and sets
    ``MFK_DEVERR_INDEX`` in ``device_status()``."""
    op = "embedding_grad"
    _require(grad, op, "grad", 1, at_least=True)
    index = _ids(op, ids, grad)
    if tuple(grad.shape[:-1]) != tuple(ids.shape):
        raise ValueError(f"{op}: grad {tuple(grad.shape)} does not fit ids {tuple(ids.shape)}")
    if not isinstance(rows, int) or isinstance(rows, bool) or rows < 0:
        raise ValueError(f"{op}: rows must be a whole number of at least 0, got {rows!r}")
    if padding is not None and (not isinstance(padding, int) or isinstance(padding, bool)):
        raise ValueError(f"{op}: padding must be a whole number, got {padding!r}")
    if padding is not None and not 0 <= padding < rows:
        raise ValueError(f"{op}: padding {padding} is outside the table of {rows} rows")
    _kernel_for(op, grad)
    d, n = grad.shape[-1], index.numel()
    if rows == 0 and n and d:
        raise ValueError(f"{op}: the table has no rows")
    g = _rows_of(grad, n, d)
    if d > 1 and g.stride(1) != 1:
        g = contiguous(g)
    out = grad.new_empty((rows, d))
    _run(grad.device, op, _lib.lib().mfk_embedding_grad_f32, _ptr(g), n, d,
         g.stride(0) if n > 1 else max(d, 1), _ptr(index), index.element_size(), rows,
         float(scale), -1 if padding is None else padding, _ptr(out), max(d, 1))
    return out
