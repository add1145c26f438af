"""Distillation from a teacher's top logits: the loss by which a converted model
is tuned against its float original.

    l = T^2 sum_i p_i (log p_i - log q_i)

p is the softmax of the logits that the teacher gives for a row (its largest, with
their places in the vocabulary), q that of the student's whole row, both at
temperature T; T^2 keeps the gradients' size whatever the temperature.
``csrc/sfb_distill.cu`` has the kernels.  No counterpart in the reference.
"""
from __future__ import annotations

from array import array

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._errors import SFShapeError, SFTypeError
from ._tensor import _FLOATS, _refuse_tangents

_INDEXES = {torch.int64: 1, torch.int32: 0}


def _check(logits, teacher, index, temperature, weight, reduction):
    if reduction not in _lib.REDUCTIONS:
        raise ValueError(f"distill_loss: reduction must be one of {tuple(_lib.REDUCTIONS)}, got {reduction!r}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"distill_loss: a temperature is between 1e-6 and 1e6, got {temperature}")
    for t, name in ((logits, "logits are"), (teacher, "teacher's logits are")):
        if t.dtype not in _FLOATS:
            raise SFTypeError(f"distill_loss: the {name} {t.dtype}; float32, bfloat16 and float16 are supported")
    if index.dtype not in _INDEXES:
        raise SFTypeError(f"distill_loss: the teacher's indexes are {index.dtype}; int64 and int32 are supported")
    if not logits.is_cuda:
        raise SFShapeError(f"distill_loss: the logits must be on a CUDA device, got {logits.device}")
    if not logits.dim() or logits.shape[-1] < 1:
        raise SFShapeError(f"distill_loss: the logits have shape {tuple(logits.shape)}, expected (..., vocabulary)")
    rows = logits.shape[:-1]
    if teacher.shape != index.shape or not teacher.dim() or teacher.shape[:-1] != rows:
        raise SFShapeError(f"distill_loss: the teacher's logits and indexes have shapes {tuple(teacher.shape)} and "
                           f"{tuple(index.shape)}; both are {(*rows, 'k')}")
    if teacher.shape[-1] > _lib.DISTILL_MOST:
        raise SFShapeError(f"distill_loss: the teacher gives {teacher.shape[-1]} entries a row, {_lib.DISTILL_MOST} at most")
    if weight is not None:
        if weight.shape != rows:
            raise SFShapeError(f"distill_loss: the rows' weights have shape {tuple(weight.shape)}, expected {tuple(rows)}")
        if weight.dtype is not torch.bool and weight.dtype not in _FLOATS:
            raise SFTypeError(f"distill_loss: the rows' weights are {weight.dtype}; bool, float32, bfloat16 and float16 are "
                              f"supported")
        if weight.requires_grad:
            raise SFTypeError("distill_loss: the rows' weights have no gradient; pass them detached")
    at = logits.get_device()
    for t, name in ((teacher, "teacher's logits"), (index, "teacher's indexes"), (weight, "rows' weights")):
        if t is not None and t.get_device() != at:
            raise SFShapeError(f"distill_loss: the {name} are on {t.device}, the logits on {logits.device}")
    if teacher.requires_grad and torch.is_grad_enabled():
        raise SFTypeError("distill_loss: the teacher's logits have no gradient; pass them detached")


def _two_strides(t):
    """(t, rows of the inner dimension, outer stride, inner stride): t's rows as at most two nested runs of rows whose
    elements are contiguous, copied where they are not."""
    V = t.shape[-1]
    if t.is_contiguous():
        return t, max(1, t.numel() // V), 0, V
    if t.stride(-1) == 1 or V == 1:
        runs = []                                     # (size, stride), the innermost first; runs that follow on join
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if runs and runs[-1][0] * runs[-1][1] == stride:
                runs[-1] = runs[-1][0] * size, runs[-1][1]
            else:
                runs.append((size, stride))
        if len(runs) <= 2:
            runs += [(1, 0)] * (2 - len(runs))
            return t, max(1, runs[0][0]), runs[1][1], runs[0][1]
    return t.contiguous(), max(1, t.numel() // V), 0, V


def _like(t):
    """An empty tensor for t's gradient: laid out as t where that wastes at most a quarter, so that the rows of both lie
    alike on 16 bytes, else compact."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return torch.empty_like(t)
    span = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    lead = t.data_ptr() % 16 // t.element_size()
    # every stride covers what lies inside it: no two elements share a place
    inside, apart = 1, True
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        apart &= s >= inside
        inside = s * (n - 1) + inside
    if not apart or 4 * span > 5 * t.numel():
        return torch.empty(t.shape, dtype=t.dtype, device=t.device)
    return torch.empty(span + lead, dtype=t.dtype, device=t.device).as_strided(t.shape, t.stride(), lead)


def _call(logits, teacher, index, weight, temperature, reduction):
    """The fields of a call but for the results; the tensors whose addresses they hold."""
    V, K = logits.shape[-1], teacher.shape[-1]
    logits, inner, so, si = _two_strides(logits)
    teacher, index = teacher.contiguous(), index.contiguous()
    w_kind = _lib.WEIGHT_NONE
    if weight is not None:
        weight = weight.contiguous()
        w_kind = _lib.WEIGHT_BYTES if weight.dtype is torch.bool else _FLOATS[weight.dtype]
    words = (_FLOATS[logits.dtype], logits.numel() // V, V, logits.data_ptr(), inner, so, si, K, teacher.data_ptr(),
             _FLOATS[teacher.dtype], K, index.data_ptr(), _INDEXES[index.dtype], K, 0 if weight is None else weight.data_ptr(),
             w_kind, _lib.REDUCTIONS[reduction], _lib.bits_of(temperature))
    return words, (logits, teacher, index, weight)


def _strides_of(grad, logits):
    """The gradient's strides by the logits' two runs of rows."""
    _, inner, so, si = _two_strides(logits)
    return (so, si) if grad.stride() == logits.stride() else (inner * logits.shape[-1], logits.shape[-1])


def _kept_size(words, keep):
    return words[1] * (4 * (words[7] + 3 & -4) + (3 if keep else 0))


def _kept_at(kept, words, keep):
    """The places of the rows' statistics and of the entries."""
    at = kept.data_ptr()
    return (at + 16 * words[1] * (words[7] + 3 & -4)) if keep else 0, at


def _forward(logits, teacher, index, weight, temperature, reduction, keep, with_grad):
    words, held = _call(logits, teacher, index, weight, temperature, reduction)
    M, logits, dev = words[1], held[0], logits.device
    mean, none = reduction == "mean", reduction == "none"
    parts = _lib.distill_parts(M) if mean else 0
    out = torch.empty(logits.shape[:-1] if none else (), dtype=torch.float32, device=dev)
    # places in one buffer: the entries and, for the backward pass, three numbers a row; then, for this call alone, the
    # rows' losses, the partial sums of the weights, the rows' weights and a counter
    kept = torch.empty(_kept_size(words, keep) + (1 if none else 2) * M + parts + 1, dtype=torch.float32, device=dev)
    grad, go, gi = None, 0, 0
    if with_grad:
        grad = _like(logits)
        go, gi = _strides_of(grad, logits)
    at = kept.data_ptr() + 4 * _kept_size(words, keep)
    rows = 0 if none else 4 * M
    _lib.distill_forward(logits.get_device(), array("q", (
        *words, 0 if none else out.data_ptr(), out.data_ptr() if none else at, at + rows, at + rows + 4 * parts,
        *_kept_at(kept, words, keep), 0 if grad is None else grad.data_ptr(), go, gi, 0, 0)))
    return out, words, held[0], kept, grad


def _gradients(ctx, g):
    logits, kept = ctx.saved_tensors
    for t, (kind, size, device) in zip((logits, kept), ctx.kept):
        if t.dtype is not kind or t.shape != size or t.device != device:
            raise (SFShapeError if t.dtype is kind else SFTypeError)(
                f"distill_loss: the backward pass kept a tensor of {kind}, {tuple(size)} on {device}; a saved-tensor hook "
                f"gave back {t.dtype}, {tuple(t.shape)} on {t.device}")
    words, strides, captured = ctx.call
    grad, ctx.grad = ctx.grad, None
    # The forward pass's gradient is the one of this call where nothing can have come between: another backward pass has
    # its own, and so has one that a graph replays without the forward pass, or one whose logits a hook laid out anew.
    if grad is not None and (_lib.capture_id(logits.get_device()) != captured or logits.stride() != strides):
        grad = None
    skip = grad is not None
    logits, inner, so, si = _two_strides(logits)
    if not skip:
        grad = _like(logits)
    g, kept = g.contiguous(), kept.contiguous()
    if kept.data_ptr() % 16:
        kept = kept.clone()
    _lib.distill_backward(logits.get_device(), array("q", (
        *words[:3], logits.data_ptr(), inner, so, si, words[7], 0, words[9], words[10], 0, words[12], words[13], 0,
        _lib.WEIGHT_NONE, *words[16:], 0, 0, 0, 0, *_kept_at(kept, words, True), grad.data_ptr(), *_strides_of(grad, logits),
        g.data_ptr(), int(skip))))
    return grad, None, None, None, None, None


# with create_graph=True: gradients that refuse to be differentiated again
_gradients_once = torch.autograd.function.once_differentiable(_gradients)


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, index, weight, temperature, reduction):
        # The gradient with the loss: the row is at hand, and a backward pass that gets a gradient of one has nothing to
        # do.  float16's waits for the scale that its loss gets, below which it would round to zero.
        with_grad = reduction != "none" and logits.dtype is not torch.float16
        loss, words, rows, kept, grad = _forward(logits, teacher, index, weight, temperature, reduction, True, with_grad)
        ctx.save_for_backward(rows, kept)
        ctx.kept = [(t.dtype, t.shape, t.device) for t in (rows, kept)]
        ctx.grad = grad
        ctx.call = words, rows.stride(), _lib.capture_id(logits.get_device()) if with_grad else 0
        return loss

    @staticmethod
    def backward(ctx, g):
        return (_gradients_once if torch.is_grad_enabled() else _gradients)(ctx, g)


def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor, *,
                 temperature: float = 1.0, row_weight=None, reduction: str = "mean") -> torch.Tensor:
    """``T^2 sum_i p_i (log p_i - log q_i)`` a row, from a teacher's top logits.

    ``logits`` (..., V): the student's, float32, bfloat16 or float16.
    ``teacher_logits`` and ``teacher_index`` (..., k), k at most 1024: what the teacher
    gives of the row, p being its softmax / T over these entries alone, and their places in
    the vocabulary (int64 or int32).  An entry is absent where its index is not in
    0 .. V - 1 (as -1) or its logit is -inf; an index given twice has the sum of both.
    ``row_weight`` (...): truth values or numbers, one a row.  A row of weight 0, or
    without entries, gives 0 whatever it holds.  ``reduction``: "mean" (over the weights
    of the rows with entries; 0 where these add up to 0), "sum", or "none" (a loss a row).
    The loss is float32, and so are all sums.  Everything is on one CUDA device; the work is
    queued on its current stream.  Differentiable once, by reverse mode, in the logits,
    whose gradient has their type; in bfloat16 and float32 it is made with a loss that is
    one number, and held from there to the backward pass."""
    if torch.compiler.is_compiling():
        return _between_graphs(logits, teacher_logits, teacher_index, temperature, row_weight, reduction)
    _check(logits, teacher_logits, teacher_index, temperature, row_weight, reduction)
    if forward_ad._current_level >= 0:
        _refuse_tangents(logits, teacher_logits, row_weight, what="distill_loss")
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillLoss.apply(logits, teacher_logits, teacher_index, row_weight, temperature, reduction)
    return _forward(logits, teacher_logits, teacher_index, row_weight, temperature, reduction, False, False)[0]


@torch.compiler.disable
def _between_graphs(logits, teacher_logits, teacher_index, temperature, row_weight, reduction):
    """A compiled training step runs the loss eagerly between its graphs."""
    return distill_loss(logits, teacher_logits, teacher_index, temperature=temperature, row_weight=row_weight,
                        reduction=reduction)
