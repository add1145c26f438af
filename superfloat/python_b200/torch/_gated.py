"""The gated feed-forward product over sf codes on the tensor cores.

    h = act(x Wg^T + bg) * (x Wu^T + bu)

What a converted transformer's gated block has before its last projection: both
weights quantized as :func:`tensor_linear`'s, both products made as one, which
reads x once, and joined where they are summed.  ``csrc/sfb_gated.cu`` and
``csrc/sfb_tensor_gemm.cu`` have the kernels.  No counterpart in the reference.
"""
from __future__ import annotations

from array import array

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._errors import SFShapeError, SFTypeError
from . import _core
from ._tensor import (_FLOATS, _TYPES, SFPackedWeight, _check_operands, _check_weight, _check_width, _refuse_tangents, _rows,
                      _rows_on16, _two_d, pack_weight)


def _check_pair(gate, up):
    if isinstance(gate, SFPackedWeight) != isinstance(up, SFPackedWeight):
        raise SFTypeError("tensor_gated: both weights are packed, or neither")
    if gate.shape != up.shape:
        raise SFShapeError(f"tensor_gated: the weights have shapes {tuple(gate.shape)} and {tuple(up.shape)}; both are (N, K)")


def _bias(t):
    if t is None:
        return None, 0, 0
    if not t.is_contiguous():
        t = t.contiguous()
    return t, t.data_ptr(), _FLOATS[t.dtype]


def _forward(x, gate, up, N, K, packed, gate_bias, up_bias, bits, wscale, act, train):
    """The result and, with ``train``, what the backward pass reads: x (None where the buffer holds a copy of it), both
    products, the buffer of codes and scales, and the places in it.  One library call, all scratch in one buffer."""
    kind = _TYPES[x.dtype]
    out = x.new_empty((*x.shape[:-1], N))
    x, ldx = _two_d(x, K)
    M, x_ptr = x.shape[0], x.data_ptr()
    Np, ldk = N + 15 & -16, K + 7 & -8
    if M <= 1:
        ldx = max(ldx, ldk) if ldx % 8 == 0 else ldk
    small = packed and M <= _lib.SMALL_ROWS and not train
    # places in one buffer, each on 256 bytes: codes, scales, the rows' maxima, x with its rows on 16 bytes
    size = scale_at = work = xpad = 0
    if not small:
        scale_at = 4 * Np * ldk + 255 & -256
        size = scale_at + (8 * Np + 255 & -256)
    gate_scale = up_scale = None
    if packed:
        (g, ldg), (u, ldu) = _rows(gate.codes, K), _rows(up.codes, K)
        w_kind, gate_scale, up_scale = _lib.I8, gate.scale.contiguous(), up.scale.contiguous()
    else:
        (g, ldg), (u, ldu) = _rows(gate, K), _rows(up, K)
        w_kind = _FLOATS[g.dtype]
        if wscale == "per_tensor":
            work = size
            size += 8 * N + 255 & -256
    pad = bool(x_ptr % 16 or ldx % 8)
    if pad:
        xpad = size
        size += 2 * M * ldk
    buf, base = None, 0
    if size:
        buf = x.new_empty(size, dtype=torch.uint8)
        base = buf.data_ptr()
    z = x.new_empty((M, 2 * Np), dtype=torch.float32) if train else None
    gate_bias, gb, gb_kind = _bias(gate_bias)
    up_bias, ub, ub_kind = _bias(up_bias)
    _lib.gated_forward(x.get_device(), array("q", (
        kind, bits, act, M, N, K, x_ptr, ldx, base + xpad, ldk, g.data_ptr(), u.data_ptr(), ldg, ldu, w_kind,
        wscale == "per_channel", gate_scale.data_ptr() if packed else 0, up_scale.data_ptr() if packed else 0,
        0 if small else base, ldk, 0 if small else base + scale_at, gb, ub, gb_kind, ub_kind, out.data_ptr(), N,
        0 if z is None else z.data_ptr(), 2 * Np, base + work, 0, 0, 0, 0, 0, 0, 0, 0, 0)))
    if not train:
        return out
    return out, (None if pad else x), z, buf, (M, N, K, xpad, scale_at)


def _refuse_kept(t, dtype, shape, device):
    error = SFShapeError if t.dtype is dtype else SFTypeError
    raise error(f"tensor_gated: the backward pass kept a tensor of {dtype}, {tuple(shape)} on {device}; a saved-tensor hook "
                f"gave back {t.dtype}, {tuple(t.shape)} on {t.device}")


def _gradients(ctx, grad):
    xs, z, buf = ctx.saved_tensors
    M, N, K, x_at, scale_at, shape, dt, bits, act, w_dtype, gb_dtype, ub_dtype, size, device = ctx.call
    want_x, want_g, want_u, _, want_gb, want_ub = ctx.needs_input_grad[:6]
    Np = N + 15 & -16
    dx = grad.new_empty(shape) if want_x else None
    dg = du = None
    if want_g and want_u:
        # one product makes both: rows of the gate's, and of the other's Np on (each counts its own changes: a view of
        # `both` would count the other's too, and a graph that has saved one refuse what was done to the other)
        both = grad.new_empty((2 * Np, K), dtype=w_dtype)
        dg, du = both[:N].data, both[Np:Np + N].data
    elif want_g or want_u:
        dw = grad.new_empty((N, K), dtype=w_dtype)
        dg, du = (dw, None) if want_g else (None, dw)
    dgb = grad.new_empty((N,), dtype=gb_dtype) if want_gb else None
    dub = grad.new_empty((N,), dtype=ub_dtype) if want_ub else None
    if M == 0:
        for t in (dg, du, dgb, dub):
            if t is not None:
                t.zero_()
        return dx, dg, du, None, dgb, dub, None, None, None
    # saved-tensor hooks (activation offloading) may give back copies of another layout
    if buf.dtype is not torch.uint8 or buf.numel() != size or buf.device != device:
        _refuse_kept(buf, torch.uint8, (size,), device)
    if buf.data_ptr() % 16 or not buf.is_contiguous():
        buf = buf.clone()
    if z.dtype is not torch.float32 or z.shape != (M, 2 * Np) or z.device != device:
        _refuse_kept(z, torch.float32, (M, 2 * Np), device)
    if z.data_ptr() % 16 or not z.is_contiguous():
        z = z.clone(memory_format=torch.contiguous_format)
    base, ldk = buf.data_ptr(), K + 7 & -8
    if xs is None:
        x_ptr, ldx = base + x_at, ldk
    else:
        if xs.dtype is not dt or xs.shape != (M, K) or xs.device != device:
            _refuse_kept(xs, dt, (M, K), device)
        xs, ldx = _rows_on16(xs, K)
        x_ptr = xs.data_ptr()
    grad, ldy = _two_d(grad, N)
    # places in one buffer: the largest scale, dz, dz s, the biases' partial sums
    one = 4 * M * Np
    dz = 256
    dzs = dz + (one if want_g or want_u else 0)
    sums = dzs + (one if want_x else 0)
    work = buf.new_empty(sums + (_lib.gated_sums(M, N) if want_gb or want_ub else 0))
    at = work.data_ptr()
    _lib.gated_backward(buf.get_device(), array("q", (
        _TYPES[dt], bits, act, M, N, K, x_ptr, ldx, 0, 0, 0, 0, 0, 0, _FLOATS[w_dtype] if want_g or want_u else 0, 1, 0, 0,
        base, ldk, base + scale_at, 0, 0, _FLOATS[gb_dtype] if want_gb else 0, _FLOATS[ub_dtype] if want_ub else 0,
        grad.data_ptr(), ldy, z.data_ptr(), 2 * Np, at + sums, at, at + dz, at + dzs, 2 * Np,
        0 if dx is None else dx.data_ptr(), 0 if dg is None else dg.data_ptr(), 0 if du is None else du.data_ptr(),
        0 if dgb is None else dgb.data_ptr(), 0 if dub is None else dub.data_ptr())))
    return dx, dg, du, None, dgb, dub, None, None, None


# with create_graph=True: gradients that refuse to be differentiated again
_gradients_once = torch.autograd.function.once_differentiable(_gradients)


class _TensorGated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, packed, gate_bias, up_bias, bits, wscale, act):
        N, K = (packed[0] if packed else gate).shape
        y, xs, z, buf, layout = _forward(x, *(packed or (gate, up)), N, K, bool(packed), gate_bias, up_bias, bits, wscale, act,
                                         True)
        ctx.save_for_backward(xs, z, buf)
        ctx.call = (*layout, x.shape, x.dtype, bits, act, None if packed else gate.dtype,
                    None if gate_bias is None else gate_bias.dtype, None if up_bias is None else up_bias.dtype, buf.numel(),
                    buf.device)
        return y

    @staticmethod
    def backward(ctx, g):
        return (_gradients_once if torch.is_grad_enabled() else _gradients)(ctx, g)


def tensor_gated(x: torch.Tensor, gate, up, gate_bias=None, up_bias=None, *, activation: str | None = "silu", dtype="sf8",
                 scale: str = "per_channel") -> torch.Tensor:
    """``act(x Wg^T + gate_bias) * (x Wu^T + up_bias)`` over sf4..sf8 codes on the tensor cores.

    ``x`` (..., K): bfloat16 or float16, the result's type.  ``gate`` and ``up``:
    two (N, K) float tensors of one type, quantized in the call to ``dtype`` codes with
    a ``scale`` "per_channel" or "per_tensor" (one for each of the two; their gradients
    are straight through), or two :class:`SFPackedWeight` of one width (``dtype`` and
    ``scale`` are then their own).  ``gate_bias`` and ``up_bias`` (N,): float32 or 16 bits, or
    None.  ``activation``: "silu", "gelu" (erf), "gelu_tanh", "relu" or None.
    Sums and both products are float32; the result is rounded once.  Everything is on one CUDA
    device; the work is queued on its current stream.  Differentiable once, by reverse
    mode, in x, float weights and the biases; the backward pass keeps x, the codes and both
    products (in float32), and rounds the products' gradients to x's type, as they are
    operands of the weights' and x's gradients."""
    if torch.compiler.is_compiling():
        return _between_graphs(x, gate, up, gate_bias, up_bias, activation, dtype, scale)
    _check_pair(gate, up)
    packed = None
    if isinstance(gate, SFPackedWeight):
        packed, gate, up = (gate, up), None, None
        bits = packed[0].bits
        if packed[1].bits != bits:
            raise SFTypeError(f"tensor_gated: the weights are sf{bits} and sf{packed[1].bits}; both have one width")
        (N, K), index = packed[0].shape, packed[0].codes.get_device()
        second, tensors = packed[1].codes, (packed[0].scale, packed[1].scale)
    else:
        from .._array import resolve_dtype
        bits = resolve_dtype(dtype).bits
        _check_width(bits)
        _core.check_args(bits, scale)
        _check_weight(gate)
        _check_weight(up)
        if gate.dtype != up.dtype:
            raise SFTypeError(f"tensor_gated: the weights are {gate.dtype} and {up.dtype}; both have one type")
        (N, K), index = gate.shape, gate.get_device()
        second, tensors = up, (gate, up)
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, *tensors, gate_bias, up_bias, what="tensor_gated")
    _check_operands(x, packed[0] if packed else None, N, K, index, gate_bias, activation, None)
    if second.get_device() != index:
        raise SFShapeError("tensor_gated: both weights are on one CUDA device")
    if up_bias is not None:
        _check_operands(x, packed[0] if packed else None, N, K, index, up_bias, activation, None)
    act = _lib.ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or (packed is None and (gate.requires_grad or up.requires_grad))
                                    or (gate_bias is not None and gate_bias.requires_grad)
                                    or (up_bias is not None and up_bias.requires_grad)):
        return _TensorGated.apply(x, gate, up, packed, gate_bias, up_bias, bits, scale, act)
    if packed is None and x.numel() <= _lib.SMALL_ROWS * K:
        # few rows: int8 codes are half the bytes of the product's operand, and the product reads them as they are
        packed = pack_weight(gate, bits, scale), pack_weight(up, bits, scale)
    return _forward(x, *(packed or (gate, up)), N, K, bool(packed), gate_bias, up_bias, bits, scale, act, False)


@torch.compiler.disable
def _between_graphs(x, gate, up, gate_bias, up_bias, activation, dtype, scale):
    """A compiled model runs the product eagerly between its graphs."""
    return tensor_gated(x, gate, up, gate_bias, up_bias, activation=activation, dtype=dtype, scale=scale)
