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

from dataclasses import dataclass

import torch

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


def _up8(n: int) -> int:
    return -(-n // 8) * 8


def _ptr(t):
    return None if t is None else t.data_ptr()


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


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t (2-D) with its rows contiguous, one after another."""
    if t.shape[0] <= 1 and t.stride(1) == 1:
        return t
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _operand(t: torch.Tensor) -> torch.Tensor:
    """t (2-D) as an operand of the products: rows on 16-byte boundaries."""
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1]:
        return t
    out = torch.empty(t.shape[0], _up8(t.shape[1]), dtype=t.dtype, device=t.device)[:, :t.shape[1]]
    return out.copy_(t)


def _quantize(w, bits, wscale, dtype, stream):
    """(codes, scale): int8 codes for a dtype of None, else the product's operand."""
    N, K = w.shape
    w = _rows(w)
    if dtype is None:
        codes, kind = torch.empty(N, K, dtype=torch.int8, device=w.device), _lib.I8
    else:
        codes, kind = torch.empty(N, _up8(K), dtype=dtype, device=w.device)[:, :K], _TYPES[dtype]
    both = torch.empty(2, N, dtype=torch.float32, device=w.device)       # the scales; the rows' maxima
    _lib.code_quantize(w.data_ptr(), _FLOATS[w.dtype], N, K, max(w.stride(0), K), bits, wscale == "per_channel",
                       codes.data_ptr(), max(codes.stride(0), K), kind, both[0].data_ptr(), both[1].data_ptr(), stream)
    return codes, both[0]


@torch.no_grad()
def pack_weight(weight: torch.Tensor, dtype="sf8", scale: str = "per_channel") -> SFPackedWeight:
    """A float weight (N, K) as sf codes, once, for the calls that share it.
    ``scale``: "per_channel" or "per_tensor".  The scale is max|w| / max(sf) and
    the codes are rounded to nearest, ties to even, as the other modes quantize a
    weight; a row that holds a NaN or an infinity has it as its scale."""
    from .._array import resolve_dtype
    bits = resolve_dtype(dtype).bits
    _check_width(bits)
    _core.check_args(bits, scale)
    weight = weight.detach()
    _check_weight(weight)
    with _lib.on_device(weight.get_device()) as d:
        if weight.numel() == 0:
            raise SFShapeError(f"a weight has at least one element, got {tuple(weight.shape)}")
        return SFPackedWeight(*_quantize(weight, bits, scale, None, d.stream), bits)


def _expand(packed: SFPackedWeight, dtype, stream):
    N, K = packed.shape
    codes = _rows(packed.codes)
    out = torch.empty(N, _up8(K), dtype=dtype, device=codes.device)[:, :K]
    _lib.code_expand(codes.data_ptr(), N, K, max(codes.stride(0), K), out.data_ptr(), max(out.stride(0), K),
                     _TYPES[dtype], stream)
    return out


def _forward(x, codes, scale, bits, bias, act, residual, keep_z, stream):
    """(y, z) of operands laid out as the product takes them."""
    (M, K), N = x.shape, codes.shape[0]
    y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    z = torch.empty(M, N, dtype=torch.float16, device=x.device) if keep_z else None
    if y.numel():
        _lib.tensor_linear(_TYPES[x.dtype], x.data_ptr(), max(x.stride(0), _up8(K)), codes.data_ptr(),
                           max(codes.stride(0), _up8(K)), scale.data_ptr(), bits, _ptr(bias),
                           0 if bias is None else _FLOATS[bias.dtype], act, _ptr(residual),
                           0 if residual is None else max(residual.stride(0), N), y.data_ptr(), N, _ptr(z), N, M, N,
                           K, stream)
    return y, z


def _check_operands(x, weight, bias, activation, residual):
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(_lib.ACTIVATIONS)}, got {activation!r}")
    if x.dtype not in _TYPES:
        raise SFTypeError(f"the input is {x.dtype}: the tensor cores take bfloat16 or float16 (accumulate=\"chain\" "
                          f"and \"wide\" take float32)")
    if x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise SFShapeError(f"the input has shape {tuple(x.shape)}, the weight expects {weight.shape[1]} features")
    if weight.shape[1] < 1 or weight.shape[0] < 1:
        raise SFShapeError(f"a weight has at least one row and one column, got {tuple(weight.shape)}")
    device = weight.codes.device if isinstance(weight, SFPackedWeight) else weight.device
    N = weight.shape[0]
    for name, t in (("input", x), ("bias", bias), ("residual", residual)):
        if t is not None and (t.device != device or not t.is_cuda):
            raise SFShapeError(f"the {name} is on {t.device}, the weight on {device}; both must be on one CUDA device")
    if bias is not None:
        if bias.shape != (N,):
            raise SFShapeError(f"the bias has shape {tuple(bias.shape)}, expected ({N},)")
        if bias.dtype not in _FLOATS:
            raise SFTypeError(f"the bias is {bias.dtype}; float32, bfloat16 and float16 are supported")
    if residual is not None:
        if residual.shape != (*x.shape[:-1], N):
            raise SFShapeError(f"the residual has shape {tuple(residual.shape)}, expected {(*x.shape[:-1], N)}")
        if residual.dtype != x.dtype:
            raise SFTypeError(f"the residual is {residual.dtype}, the input {x.dtype}")


def _backward(g, x, codes, scale, z, bits, act, top, want_x, want_w, w_dtype, want_b, b_dtype, stream):
    """Gradients (x, weight, bias) from the output's, all 2-D."""
    (M, K), N = x.shape, codes.shape[0]
    kind, dev = _TYPES[x.dtype], x.device
    g = _rows(g)
    dx = dw = db = None
    # per-tensor scales: top is that scale and dz s / top = dz, one operand for both products
    one_scale = top is not None and top.data_ptr() == scale.data_ptr()
    direct = act == 0 and g.data_ptr() % 16 == 0 and g.stride(0) % 8 == 0 and g.stride(0) >= N
    need_dz = (want_w or (want_x and one_scale)) and not direct
    need_dzs = want_x and not one_scale
    ldd = _up8(N)
    dz = torch.empty(M, ldd, dtype=x.dtype, device=dev)[:, :N] if need_dz else None
    dzs = torch.empty(M, ldd, dtype=x.dtype, device=dev)[:, :N] if need_dzs else None
    if want_b:
        db = torch.empty(N, dtype=b_dtype, device=dev)
    if M and (need_dz or need_dzs or want_b):
        work = torch.empty(_lib.slope_workspace(M, N), dtype=torch.uint8, device=dev) if want_b else None
        _lib.slope(kind, act, g.data_ptr(), max(g.stride(0), N), _ptr(z), N, M, N, scale.data_ptr(), bits, _ptr(top),
                   _ptr(dz), _ptr(dzs), ldd, _ptr(db), _FLOATS[b_dtype] if want_b else 0, _ptr(work), stream)
    elif want_b:
        db.zero_()
    if direct:
        dz = g
    if want_x:
        d = dz if one_scale else dzs
        dx = torch.empty(M, K, dtype=x.dtype, device=dev)
        if M:
            _lib.tensor_grad_x(kind, d.data_ptr(), max(d.stride(0), ldd), codes.data_ptr(),
                               max(codes.stride(0), _up8(K)), _ptr(top), bits, dx.data_ptr(), K, M, N, K, stream)
    if want_w:
        dw = torch.empty(N, K, dtype=w_dtype, device=dev)
        if M:
            _lib.tensor_grad_w(kind, dz.data_ptr(), max(dz.stride(0), ldd), x.data_ptr(), max(x.stride(0), _up8(K)),
                               dw.data_ptr(), _FLOATS[w_dtype], K, M, N, K, stream)
        else:
            dw.zero_()
    return dx, dw, db


class _TensorLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, packed, bias, residual, bits, wscale, act):
        with _lib.on_device(x.get_device()) as d:
            ctx.lead, N = x.shape[:-1], (packed or weight).shape[0]
            xa = _operand(x.detach().reshape(-1, x.shape[-1]))
            if packed is None:
                codes, scale = _quantize(weight.detach(), bits, wscale, x.dtype, d.stream)
            else:
                codes, scale = _expand(packed, x.dtype, d.stream), packed.scale.contiguous()
            r = None if residual is None else _rows(residual.detach().reshape(-1, N))
            b = None if bias is None else bias.detach().contiguous()
            y, z = _forward(xa, codes, scale, bits, b, act, r, act != 0, d.stream)
        ctx.save_for_backward(xa, codes, scale, z)
        ctx.bits, ctx.act = bits, act
        ctx.wscale = wscale if packed is None else "per_channel"
        ctx.w_dtype = None if packed is not None else weight.dtype
        ctx.b_dtype = None if bias is None else bias.dtype
        return y.view(*ctx.lead, N)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        xa, codes, scale, z = ctx.saved_tensors
        want_x, want_w, _, want_b, want_r = ctx.needs_input_grad[:5]
        with _lib.on_device(xa.get_device()) as d:
            top = None
            if want_x and ctx.wscale == "per_tensor":
                top = scale[:1]
            elif want_x and xa.dtype == torch.float16:
                # dz s would leave fp16's range where the scales are small: s / max s is within it
                top = scale.amax().view(1)
            dx, dw, db = _backward(g.reshape(-1, codes.shape[0]), xa, codes, scale, z, ctx.bits, ctx.act, top, want_x,
                                   want_w, ctx.w_dtype, want_b, ctx.b_dtype, d.stream)
        if dx is not None:
            dx = dx.view(*ctx.lead, xa.shape[1])
        return dx, dw, None, db, g if want_r else None, None, None, None


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
    device; the work is queued on its current stream.  Differentiable once, in
    x, a float weight, bias and residual."""
    packed = weight if isinstance(weight, SFPackedWeight) else None
    if packed is None:
        from .._array import resolve_dtype
        bits = resolve_dtype(dtype).bits
        _check_width(bits)
        _core.check_args(bits, scale)
        _check_weight(weight)
    else:
        bits = packed.bits
    _check_operands(x, weight, bias, activation, residual)
    act = _lib.ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in
                                       (x, None if packed else weight, bias, residual)):
        return _TensorLinear.apply(x, None if packed else weight, packed, bias, residual, bits, scale, act)
    return _no_grad(x, weight, packed, bias, residual, bits, scale, act)


def _no_grad(x, weight, packed, bias, residual, bits, wscale, act):
    N, K = weight.shape
    with _lib.on_device(x.get_device()) as d:
        xa = _operand(x.detach().reshape(-1, K))
        M = xa.shape[0]
        small = M <= _lib.SMALL_ROWS
        if packed is None:
            codes, scale = _quantize(weight.detach(), bits, wscale, None if small else x.dtype, d.stream)
        elif small:
            codes, scale = _rows(packed.codes), packed.scale.contiguous()
        else:
            codes, scale = _expand(packed, x.dtype, d.stream), packed.scale.contiguous()
        r = None if residual is None else _rows(residual.detach().reshape(-1, N))
        b = None if bias is None else bias.detach().contiguous()
        if small:
            y = torch.empty(M, N, dtype=x.dtype, device=x.device)
            _lib.tensor_linear_small(_TYPES[x.dtype], xa.data_ptr(), max(xa.stride(0), _up8(K)), codes.data_ptr(),
                                     max(codes.stride(0), K), scale.data_ptr(), bits, _ptr(b),
                                     0 if b is None else _FLOATS[b.dtype], act, _ptr(r),
                                     0 if r is None else max(r.stride(0), N), y.data_ptr(), N, M, N, K, d.stream)
        else:
            y, _ = _forward(xa, codes, scale, bits, b, act, r, False, d.stream)
    return y.view(*x.shape[:-1], N)


def tensor_failures() -> int:
    """How many CTAs of the tensor-core products have given up a bounded wait on
    the current device since the library was loaded; the outputs of such a CTA
    are NaN.  Waits for the device."""
    _lib.ensure_current(torch.cuda.current_device())
    return _lib.tensor_failures()
