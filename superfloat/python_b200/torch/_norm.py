"""Layer norm over the last dimension, forward and backward, on the B200.

    y = (x - mean) / sqrt(var + eps) * weight + bias

What stands before the projections of a converted transformer: the tensor-core
layers take bfloat16 or float16 and so does this, with its statistics in
float32.  ``csrc/sfb_norm.cu`` has the kernels.  No counterpart in the reference.
"""
from __future__ import annotations

from array import array

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._errors import SFShapeError, SFTypeError
from ._tensor import _FLOATS, _refuse_tangents, _two_d


def _check(x, weight, bias, eps):
    if x.dtype not in _FLOATS:
        raise SFTypeError(f"layer_norm: the input is {x.dtype}; float32, bfloat16 and float16 are supported")
    if not x.is_cuda:
        raise SFShapeError(f"layer_norm: the input must be on a CUDA device, got {x.device}")
    shape, at = x.shape, x.get_device()
    if not shape or not 1 <= shape[-1] <= _lib.NORM_MOST:
        raise SFShapeError(f"layer_norm: the last dimension has 1 to {_lib.NORM_MOST} features, got {tuple(shape)}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.shape != shape[-1:]:
            raise SFShapeError(f"layer_norm: the {name} has shape {tuple(t.shape)}, expected ({x.shape[-1]},)")
        if t.dtype not in _FLOATS:
            raise SFTypeError(f"layer_norm: the {name} is {t.dtype}; float32, bfloat16 and float16 are supported")
        if t.get_device() != at:
            raise SFShapeError(f"layer_norm: the {name} is on {t.device}, the input on {x.device}")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")


def _flat(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _address(t):
    return (0, 0) if t is None else (t.data_ptr(), _FLOATS[t.dtype])


def _forward(x, weight, bias, eps, keep):
    D = x.shape[-1]
    y = torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
    x, ldx = _two_d(x, D)
    M, index = x.shape[0], x.get_device()
    stats = x.new_empty((M, 2), dtype=torch.float32) if keep else None
    weight, bias = _flat(weight), _flat(bias)
    _lib.norm_forward(index, array("q", (
        _FLOATS[x.dtype], M, D, x.data_ptr(), ldx, *_address(weight), *_address(bias), _lib.bits_of(eps), y.data_ptr(), D,
        stats.data_ptr() if keep else 0, 0, 0, 0, 0, 0)))
    return y, x, stats


def _gradients(ctx, g):
    x, weight, stats = ctx.saved_tensors
    M, D, dtype, w_dtype, b_dtype, device, shape = ctx.call
    want_x, want_w, want_b = ctx.needs_input_grad[:3]
    dx = g.new_empty(shape) if want_x else None
    dw = g.new_empty((D,), dtype=w_dtype) if want_w else None
    db = g.new_empty((D,), dtype=b_dtype) if want_b else None
    if M == 0:
        for t in (dw, db):
            if t is not None:
                t.zero_()
        return dx, dw, db, None
    # saved-tensor hooks (activation offloading) may give back copies of another layout
    for t, kind, size in ((x, dtype, (M, D)), (weight, w_dtype, (D,)), (stats, torch.float32, (M, 2))):
        if t is not None and (t.dtype is not kind or t.shape != size or t.device != device):
            raise (SFShapeError if t.dtype is kind else SFTypeError)(
                f"layer_norm: the backward pass kept a tensor of {kind}, {size} on {device}; a saved-tensor hook gave back "
                f"{t.dtype}, {tuple(t.shape)} on {t.device}")
    x, ldx = _two_d(x, D)
    g, ldg = _two_d(g, D)
    weight, stats = _flat(weight), _flat(stats)
    if stats.data_ptr() % 8:
        stats = stats.clone()
    work = g.new_empty(_lib.norm_work(M, D), dtype=torch.uint8) if want_w or want_b else None
    w_ptr, w_kind = _address(weight)
    _lib.norm_backward(x.get_device(), array("q", (
        _FLOATS[dtype], M, D, x.data_ptr(), ldx, w_ptr, w_kind, 0, _FLOATS[b_dtype] if want_b else 0, 0, g.data_ptr(), ldg,
        stats.data_ptr(), dx.data_ptr() if want_x else 0, D, dw.data_ptr() if want_w else 0, db.data_ptr() if want_b else 0,
        0 if work is None else work.data_ptr())))
    return dx, dw, db, None


# with create_graph=True: gradients that refuse to be differentiated again
_gradients_once = torch.autograd.function.once_differentiable(_gradients)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, rows, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(rows, weight, stats)
        ctx.call = (*rows.shape, x.dtype, None if weight is None else weight.dtype, None if bias is None else bias.dtype,
                    x.device, x.shape)
        return y

    @staticmethod
    def backward(ctx, g):
        return (_gradients_once if torch.is_grad_enabled() else _gradients)(ctx, g)


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    ``x`` (..., D): float32, bfloat16 or float16, the result's type; D is at most
    65536.  ``weight`` and ``bias`` (D,): each of any of the three types, or None
    (one, zero).  Statistics and sums are float32; the result is rounded once.
    Everything is on one CUDA device; the work is queued on its current stream.
    Differentiable once, by reverse mode, in x, weight and bias; the backward pass
    keeps x and two numbers a row."""
    if torch.compiler.is_compiling():
        return _between_graphs(x, weight, bias, eps)
    _check(x, weight, bias, eps)
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight, bias, what="layer_norm")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]


@torch.compiler.disable
def _between_graphs(x, weight, bias, eps):
    """A compiled model runs the norm eagerly between its graphs."""
    return layer_norm(x, weight, bias, eps)
