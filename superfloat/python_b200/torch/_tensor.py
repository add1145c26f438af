"""The linear layer over sf codes on the tensor cores, with its epilogue.

    y = act(x Wq^T + bias) + residual,   Wq[n, k] = code[n, k] 2^-(N-1) scale[n]

The chain and wide modes compute a converted layer as the chip does, step by
step on integers.  This mode keeps what the conversion does to the weights
(sf4..sf8 codes and their scales) and takes the activations in bf16 or fp16,
summing in float32: what training and serving need at tensor-core speed.  It
has no counterpart in the reference.

The weight is a float tensor, quantized in the call with a straight-through
gradient, or an :class:`SFPackedWeight`, codes and scales laid out once.
``csrc/sfb_tensor_gemm.cu`` and ``csrc/sfb_tensor_codes.cu`` have the kernels.
"""
from __future__ import annotations

from array import array
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._errors import SFShapeError, SFTypeError, SFUnsupportedError
from . import _core

BITS = (4, 5, 6, 7, 8)
_TYPES = {torch.bfloat16: _lib.ELEMENT["bfloat16"], torch.float16: _lib.ELEMENT["float16"]}
_FLOATS = {**_TYPES, torch.float32: _lib.ELEMENT["float32"]}


@dataclass
class SFPackedWeight:
    """A weight as sf codes: ``codes`` (N, K) int8 in +-(2^(bits-1) - 1), rows
    contiguous, and ``scale`` (N,) float32; see :func:`pack_weight`."""

    codes: torch.Tensor
    scale: torch.Tensor
    bits: int = 8

    def __post_init__(self):
        if self.bits not in BITS:
            raise SFUnsupportedError(f"packed weights are sf4..sf8, got sf{self.bits}")
        if self.codes.dtype != torch.int8 or self.scale.dtype != torch.float32:
            raise SFTypeError(f"a packed weight has int8 codes and float32 scales, got {self.codes.dtype} and "
                              f"{self.scale.dtype}")
        if self.codes.dim() != 2 or self.scale.shape != self.codes.shape[:1]:
            raise SFShapeError(f"a packed weight has (N, K) codes and (N,) scales, got {tuple(self.codes.shape)} and "
                               f"{tuple(self.scale.shape)}")
        if self.codes.device != self.scale.device:
            raise SFShapeError("a packed weight's codes and scales are on one device")

    @property
    def shape(self):
        return self.codes.shape

    def dequantize(self) -> torch.Tensor:
        """The float32 weight the codes stand for."""
        return self.codes.float() * (self.scale * 2.0 ** (1 - self.bits))[:, None]


def _check_width(bits: int) -> None:
    if bits not in BITS:
        raise SFUnsupportedError(f"the tensor-core linear takes sf4..sf8, whose codes are exact in 16-bit floats; got "
                                 f"sf{bits} (accumulate=\"chain\" and \"wide\" run it)")


def _check_weight(w: torch.Tensor) -> None:
    if w.dim() != 2:
        raise SFShapeError(f"a weight has two dimensions, got {tuple(w.shape)}")
    if w.dtype not in _FLOATS:
        raise SFTypeError(f"the weight is {w.dtype}; float32, bfloat16 and float16 are supported")
    if not w.is_cuda:
        raise SFShapeError(f"the weight must be on a CUDA device, got {w.device}")
    if w.numel() == 0:
        raise SFShapeError(f"a weight has at least one row and one column, got {tuple(w.shape)}")


def _rows(t: torch.Tensor, width: int):
    """(t, row stride): t (2-D) with each row contiguous and the rows one after another."""
    ld, inner = t.stride()
    if (inner == 1 or width == 1) and (ld >= width or t.shape[0] <= 1):
        return t, max(ld, width)
    return t.contiguous(), width


def _two_d(t: torch.Tensor, width: int):
    return _rows(t if t.dim() == 2 else t.reshape(-1, width), width)


def _rows_on16(t: torch.Tensor, width: int):
    """(t, row stride): t (2-D, 16 bits) with its rows on 16 bytes, copied where they are not."""
    t, ld = _rows(t, width)
    if t.shape[0] <= 1:
        ld = width + 7 & -8
    if t.data_ptr() % 16 or ld % 8:
        ld = width + 7 & -8
        t = t.new_empty(t.shape[0], ld)[:, :width].copy_(t)
    return t, ld


@torch.no_grad()
def pack_weight(weight: torch.Tensor, dtype="sf8", scale: str = "per_channel") -> SFPackedWeight:
    """A float weight (N, K) as sf codes, once, for the calls that share it.
    ``scale``: "per_channel" or "per_tensor".  The scale is max|w| / max(sf) and
    the codes are rounded to nearest, ties to even, as the other modes quantize a
    weight; a row that holds a NaN or an infinity has it as its scale."""
    from .._array import resolve_dtype
    bits, scale_kind = resolve_dtype(dtype).bits, scale
    _check_width(bits)
    _core.check_args(bits, scale_kind)
    weight = weight.detach()
    _check_weight(weight)
    (N, K), (weight, ldw) = weight.shape, _rows(weight, weight.shape[1])
    dev = weight.device
    # rows on 16 bytes: what the few-rows product reads a row's codes in
    codes = torch.empty(N, K + 15 & -16, dtype=torch.int8, device=dev)[:, :K]
    scale, work = torch.empty(N, dtype=torch.float32, device=dev), None
    if scale_of_all := scale_kind == "per_tensor":
        work = torch.empty(N, dtype=torch.float32, device=dev)
    with _lib.on_device(weight.get_device()) as d:
        _lib.code_quantize(weight.data_ptr(), _FLOATS[weight.dtype], N, K, ldw, bits, not scale_of_all, codes.data_ptr(),
                           codes.stride(0), scale.data_ptr(), work.data_ptr() if scale_of_all else None, d.stream)
    return SFPackedWeight(codes, scale, bits)


def _check_operands(x, weight, N, K, index, bias, activation, residual):
    """The checks of a call whose weight is N x K on CUDA device ``index`` (-1: on the host)."""
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(_lib.ACTIVATIONS)}, got {activation!r}")
    dt = x.dtype
    if dt not in _TYPES:
        raise SFTypeError(f"the input is {dt}: the tensor cores take bfloat16 or float16 (accumulate=\"chain\" "
                          f"and \"wide\" take float32)")
    shape = x.shape
    if not shape or shape[-1] != K:
        raise SFShapeError(f"the input has shape {tuple(shape)}, the weight expects {K} features")
    if N < 1 or K < 1:
        raise SFShapeError(f"a weight has at least one row and one column, got {(N, K)}")
    if index < 0 or x.get_device() != index:
        raise SFShapeError(f"the input is on {x.device}, the weight on {weight.scale.device if index < 0 else index}; "
                           f"both must be on one CUDA device")
    if bias is not None:
        if bias.shape != (N,):
            raise SFShapeError(f"the bias has shape {tuple(bias.shape)}, expected ({N},)")
        if bias.dtype not in _FLOATS:
            raise SFTypeError(f"the bias is {bias.dtype}; float32, bfloat16 and float16 are supported")
        if bias.get_device() != index:
            raise SFShapeError(f"the bias is on {bias.device}, the weight on cuda:{index}")
    if residual is not None:
        if residual.shape != (*shape[:-1], N):
            raise SFShapeError(f"the residual has shape {tuple(residual.shape)}, expected {(*shape[:-1], N)}")
        if residual.dtype != dt:
            raise SFTypeError(f"the residual is {residual.dtype}, the input {dt}")
        if residual.get_device() != index:
            raise SFShapeError(f"the residual is on {residual.device}, the weight on cuda:{index}")


def _forward(x, weight, N, K, packed, bias, residual, bits, wscale, act, train):
    """The result and, with ``train``, what the backward pass reads: x (None where
    the buffer holds a copy of it), the pre-activation, the buffer of codes and
    scales, and the places in it.  One library call, all scratch in one buffer."""
    kind = _TYPES[x.dtype]
    out = x.new_empty((*x.shape[:-1], N))
    x, ldx = _two_d(x, K)
    M, x_ptr = x.shape[0], x.data_ptr()
    ldk = K + 7 & -8
    if M <= 1:
        ldx = max(ldx, ldk) if ldx % 8 == 0 else ldk
    small = packed is not None and M <= _lib.SMALL_ROWS and not train
    # places in one buffer, each on 256 bytes: codes, scales, the rows' maxima, x with its rows on 16 bytes
    codes = size = scale_at = work = xpad = 0
    if not small:
        size = 2 * N * ldk + 255 & -256
    if packed is None:
        w, ldw = _rows(weight, K)
        w_kind = _FLOATS[w.dtype]
        scale_at = size
        size += 4 * N + 255 & -256
        if wscale == "per_tensor":
            work = size
            size += 4 * N + 255 & -256
    else:
        w, ldw = _rows(packed.codes, K)
        w_kind, scale = _lib.I8, packed.scale
        if not scale.is_contiguous():
            scale = scale.contiguous()
    pad = bool(x_ptr % 16 or ldx % 8)
    if pad:
        xpad = size
        size += 2 * M * ldk
    buf, base = None, 0
    if size:
        buf = x.new_empty(size, dtype=torch.uint8)
        base = buf.data_ptr()
    z = x.new_empty((M, N), dtype=torch.float16) if train and act else None
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    r_ptr, ldr = 0, 0
    if residual is not None:
        residual, ldr = _two_d(residual, N)
        r_ptr = residual.data_ptr()
    _lib.tensor_forward(x.get_device(), array("q", (
        kind, bits, act, M, N, K, x_ptr, ldx, base + xpad, ldk, w.data_ptr(), ldw, w_kind, wscale == "per_channel",
        0 if small else base, ldk, base + scale_at if packed is None else scale.data_ptr(),
        0 if bias is None else bias.data_ptr(), 0 if bias is None else _FLOATS[bias.dtype], r_ptr, ldr,
        out.data_ptr(), N, 0 if z is None else z.data_ptr(), N, base + work, 0, 0, 0, 0, 0, 0, 0, 0)))
    if not train:
        return out
    return out, (None if pad else x), z, buf, (None if packed is None else scale), (M, N, K, xpad, scale_at)


def _refuse_kept(t, dtype, shape, device):
    error = SFShapeError if t.dtype is dtype else SFTypeError
    raise error(f"tensor_linear: the backward pass kept a tensor of {dtype}, {tuple(shape)} on {device}; a saved-tensor "
                f"hook gave back {t.dtype}, {tuple(t.shape)} on {t.device}")


def _kept(ctx):
    """What the forward pass kept: (x or None, its row stride, the pre-activation, the
    buffer, the scales).  The layouts are those of the tensors that come back, which
    saved-tensor hooks (activation offloading) may have copied: a slice of a wider
    buffer comes back compact."""
    xs, z, buf, scale = ctx.saved_tensors
    (M, N, K), dt, ldx = ctx.call[:3], ctx.call[6], 0
    size, device = ctx.buffer
    if buf.dtype is not torch.uint8 or buf.numel() != size or buf.device != device:
        _refuse_kept(buf, torch.uint8, (size,), device)
    if buf.data_ptr() % 16 or not buf.is_contiguous():
        buf = buf.clone()
    if xs is not None:
        if xs.dtype is not dt or xs.shape != (M, K) or xs.device != device:
            _refuse_kept(xs, dt, (M, K), device)
        ldx, inner = xs.stride()
        if inner != 1 or ldx % 8 or ldx < K or M == 1 or xs.data_ptr() % 16:
            xs, ldx = _rows_on16(xs, K)
    if z is not None:
        if z.dtype is not torch.float16 or z.shape != (M, N) or z.device != device:
            _refuse_kept(z, torch.float16, (M, N), device)
        if not z.is_contiguous():
            z = z.contiguous()
    if scale is not None:
        if scale.dtype is not torch.float32 or scale.shape != (N,) or scale.device != device:
            _refuse_kept(scale, torch.float32, (N,), device)
        scale = scale.contiguous()
    return xs, ldx, z, buf, scale


def _backward(g, kept, call, want_x, want_w, want_b):
    """The gradients (dx, dw, db) that are wanted, else None.  ``kept()`` gives (x or
    None, its row stride, the pre-activation, the buffer, the scales)."""
    M, N, K, x_at, scale_at, shape, dt, bits, act, per_channel, w_dtype, b_dtype = call
    dx = g.new_empty(shape) if want_x else None
    dw = g.new_empty((N, K), dtype=w_dtype) if want_w else None
    db = g.new_empty((N,), dtype=b_dtype) if want_b else None
    if M == 0:
        for t in (dw, db):
            if t is not None:
                t.zero_()
        return dx, dw, db
    xs, ldx, z, buf, scale = kept()
    g, ldg = _two_d(g, N)
    ldn, ldk = N + 7 & -8, K + 7 & -8
    # places in one buffer: the largest scale, dz, dz s, the bias's partial sums
    one = 2 * M * ldn + 255 & -256
    dz = 256
    dzs = dz + (one if want_w or not per_channel else 0)
    sums = dzs + (one if want_x and per_channel else 0)
    work = buf.new_empty(sums + (_lib.tensor_sums(M, N) if want_b else 0))
    at, base = work.data_ptr(), buf.data_ptr()
    if xs is None:
        x_ptr, ldx = base + x_at, ldk
    else:
        x_ptr = xs.data_ptr()
    _lib.tensor_backward(buf.get_device(), array("q", (
        _TYPES[dt], bits, act, M, N, K, x_ptr, ldx, 0, 0, 0, 0, _FLOATS[w_dtype] if want_w else 0,
        per_channel, base, ldk, base + scale_at if scale is None else scale.data_ptr(), 0, 0, 0, 0, g.data_ptr(),
        ldg, 0 if z is None else z.data_ptr(), N, at + sums, at, at + dz, at + dzs, ldn,
        0 if dx is None else dx.data_ptr(), 0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(),
        _FLOATS[b_dtype] if want_b else 0)))
    return dx, dw, db


def _gradients(ctx, g):
    want_x, want_w, _, want_b, want_r = ctx.needs_input_grad[:5]
    gr = g if want_r else None
    if not (want_x or want_w or want_b):
        return None, None, None, None, gr, None, None, None
    dx, dw, db = _backward(g, lambda: _kept(ctx), ctx.call, want_x, want_w, want_b)
    return dx, dw, None, db, gr, None, None, None


@torch.no_grad()
def plain_gradients(g, x, weight, bias, bits, wscale, want_x, want_w, want_b):
    """(dx, dw, db), None where not wanted, of the layer without activation and residual
    from its own inputs: the weight's codes are made again (a forward pass of no rows)."""
    _check_weight(weight)
    N, K = weight.shape
    _check_operands(x, None, N, K, weight.get_device(), bias, None, None)
    if g.shape != (*x.shape[:-1], N) or g.dtype != x.dtype or g.device != x.device:
        raise SFShapeError(f"the result's gradient is {g.dtype}, {tuple(g.shape)} on {g.device}; expected {x.dtype}, "
                           f"{(*x.shape[:-1], N)} on {x.device}")
    if want_b and bias is None:
        raise SFShapeError("there is no bias to have a gradient")
    *_, buf, scale, layout = _forward(x.new_empty((0, K)), weight, N, K, None, None, None, bits, wscale, 0, True)
    rows = x if x.dim() == 2 else x.reshape(-1, K)
    call = (rows.shape[0], *layout[1:], x.shape, x.dtype, bits, 0, wscale == "per_channel", weight.dtype,
            None if bias is None else bias.dtype)
    return _backward(g, lambda: (*_rows_on16(rows, K), None, buf, scale), call, want_x, want_w, want_b)


# with create_graph=True: gradients that refuse to be differentiated again
_gradients_once = torch.autograd.function.once_differentiable(_gradients)


class _TensorLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, packed, bias, residual, bits, wscale, act):
        N, K = (packed or weight).shape
        y, xs, z, buf, scale, layout = _forward(x, weight, N, K, packed, bias, residual, bits, wscale, act, True)
        ctx.save_for_backward(xs, z, buf, scale)
        ctx.buffer = buf.numel(), buf.device
        ctx.call = (*layout, x.shape, x.dtype, bits, act, packed is not None or wscale == "per_channel",
                    None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    def backward(ctx, g):
        # (the wrapper alone takes 5 us of a call)
        return (_gradients_once if torch.is_grad_enabled() else _gradients)(ctx, g)


def _refuse_tangents(*tensors) -> None:
    """Within a dual level: a tangent would be dropped, as the layer has no rule for it."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise SFUnsupportedError("tensor_linear has no forward-mode derivative; its gradients are reverse mode")


def tensor_linear(x: torch.Tensor, weight, bias=None, *, activation: str | None = None, residual=None, dtype="sf8",
                  scale: str = "per_channel") -> torch.Tensor:
    """``act(x Wq^T + bias) + residual`` over sf4..sf8 codes on the tensor cores.

    ``x`` (..., K) and ``residual`` (..., N): bfloat16 or float16, the result's
    type.  ``weight``: an (N, K) float tensor, quantized in the call to
    ``dtype`` codes with a ``scale`` "per_channel" or "per_tensor" (its gradient
    is straight through), or an :class:`SFPackedWeight` (``dtype`` and ``scale``
    are then the weight's own).  ``bias`` (N,): float32 or 16 bits.
    ``activation``: None, "relu", "gelu" (erf), "gelu_tanh" or "silu".
    Sums are float32; the result is rounded once.  Everything is on one CUDA
    device; the work is queued on its current stream.  Differentiable once, by
    reverse mode, in x, a float weight, bias and residual; the backward pass keeps
    x, the codes and the pre-activation (in fp16), and rounds the pre-activation's
    gradient to x's type, as it is an operand of the weight's and x's gradients."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight.scale if isinstance(weight, SFPackedWeight) else weight, bias, residual)
    if isinstance(weight, SFPackedWeight):
        packed, weight = weight, None
        (N, K), bits, index = packed.codes.shape, packed.bits, packed.codes.get_device()
    else:
        from .._array import resolve_dtype
        packed, bits = None, resolve_dtype(dtype).bits
        _check_width(bits)
        _core.check_args(bits, scale)
        _check_weight(weight)
        (N, K), index = weight.shape, weight.get_device()
    _check_operands(x, packed, N, K, index, bias, activation, residual)
    act = _lib.ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or (packed is None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _TensorLinear.apply(x, weight, packed, bias, residual, bits, scale, act)
    if packed is None and x.numel() <= _lib.SMALL_ROWS * K:
        # few rows: int8 codes are half the bytes of the product's operand, and the product reads them as they are
        packed = pack_weight(weight, bits, scale)
    return _forward(x, weight, N, K, packed, bias, residual, bits, scale, act, False)


def tensor_failures() -> int:
    """How many CTAs of the tensor-core products have given up a bounded wait on
    the current device since the library was loaded; the outputs of such a CTA
    are NaN.  Waits for the device."""
    _lib.ensure_current(torch.cuda.current_device())
    return _lib.tensor_failures()
