"""SF layers and model conversion: SFConfig, SFLinear, SFHFConv1D, SFConv2d,
convert, ConversionReport, find_lm_heads (the reference's
src/sf/torch/_modules.py:18-537, chain accumulation).

``convert`` swaps ``nn.Linear``, ``nn.Conv2d`` (groups=1, zero padding) and
Hugging Face's ``Conv1D`` (GPT-2) for SF layers that keep the source layer's
own parameter objects; each SF layer's forward is one ``sf::linear`` op run by
libsfb200.  Layers it cannot convert are listed in the report with the
reason and run as they were.
"""
from __future__ import annotations

import copy
import inspect
from dataclasses import dataclass, field

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.overrides import TorchFunctionMode

from . import _core, _gated, _norm, _tensor
from ._ops import call_linear


def _bits_of(dtype) -> int:
    from .._array import resolve_dtype
    return resolve_dtype(dtype).bits


@dataclass
class SFConfig:
    """How an SF layer computes: width, weight scale ("per_tensor" |
    "per_channel"), headroom ("bound": no saturation, provable | "none").
    ``accumulate``: "chain" and "wide" compute as the chip does; "tensor" takes
    the weights' sf4..sf8 codes to the tensor cores, with bfloat16 or float16
    activations and float32 sums (headroom and shift do not apply)."""

    bits: int = 16
    scale: str = "per_tensor"
    headroom: str = "bound"
    accumulate: str = "chain"
    shift: int | None = None

    def __post_init__(self):
        _core.check_args(self.bits, self.scale, self.headroom, self.accumulate)
        if self.accumulate == "tensor":
            _tensor._check_width(self.bits)
        if self.shift is not None:
            if self.accumulate != "wide":
                raise ValueError("shift= only applies to accumulate=\"wide\"")
            if isinstance(self.shift, bool) or not isinstance(self.shift, int):
                raise TypeError(f"shift must be an int, got {type(self.shift).__name__}")
            if not -32 <= self.shift <= 31:
                raise ValueError(f"shift must be between -32 and 31, got {self.shift}")

    @property
    def dtype_name(self) -> str:
        return f"sf{self.bits}"

    def describe(self) -> str:
        if self.accumulate == "wide":
            return f"dtype={self.dtype_name}, accumulate=wide" + ("" if self.shift is None else f", shift={self.shift}")
        if self.accumulate == "tensor":
            return f"dtype={self.dtype_name}, scale={self.scale}, accumulate=tensor"
        return f"dtype={self.dtype_name}, scale={self.scale}, headroom={self.headroom}"


class SFLinear(nn.Module):
    """``nn.Linear`` with SF arithmetic: the float parameters stay (training
    works through the straight-through gradient); every forward quantizes and
    runs the SF chain on the B200."""

    def __init__(self, in_features, out_features, bias=True, *, dtype="sf16", scale="per_tensor",
                 headroom="bound", accumulate="chain", shift=None, name="", device=None, param_dtype=None):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.sf = SFConfig(_bits_of(dtype), scale, headroom, accumulate, shift)
        self.sf_name = name or f"linear_{id(self):x}"
        ref = nn.Linear(in_features, out_features, bias, device=device, dtype=param_dtype)
        self.weight = ref.weight
        self.bias = ref.bias

    @classmethod
    def from_float(cls, m: nn.Linear, name: str, cfg: SFConfig) -> "SFLinear":
        """Wrap ``m``'s own parameter objects (an optimizer built before the
        conversion keeps working) and its training state."""
        new = cls.__new__(cls)
        nn.Module.__init__(new)
        new.in_features, new.out_features = m.in_features, m.out_features
        new.sf = cfg
        new.sf_name = name or f"linear_{id(new):x}"
        new.weight = m.weight
        new.bias = m.bias
        new.train(m.training)
        return new

    def forward(self, x):
        return call_linear(x, self.weight, self.bias, self.sf, self.sf_name)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, {self.sf.describe()}, name={self.sf_name!r}")


def is_hf_conv1d(m: nn.Module) -> bool:
    """Hugging Face's ``Conv1D``: a linear layer whose weight is stored
    ``(in, out)``, recognised by name and attributes (transformers is never
    imported)."""
    w = getattr(m, "weight", None)
    return (type(m).__name__ == "Conv1D" and isinstance(getattr(m, "nf", None), int)
            and isinstance(getattr(m, "nx", None), int) and w is not None and hasattr(w, "shape")
            and tuple(w.shape) == (m.nx, m.nf))


class SFHFConv1D(nn.Module):
    """Hugging Face ``Conv1D`` with SF arithmetic: a linear on ``weight.t()``;
    the weight keeps its ``(in, out)`` layout and is the source's parameter."""

    def __init__(self, conv: nn.Module, name: str, cfg: SFConfig):
        super().__init__()
        if not is_hf_conv1d(conv):
            raise ValueError("not a Hugging Face Conv1D")
        self.nf, self.nx = conv.nf, conv.nx
        self.sf = cfg
        self.sf_name = name
        self.weight = conv.weight
        self.bias = conv.bias
        self.train(conv.training)

    def forward(self, x):
        return call_linear(x, self.weight.t(), self.bias, self.sf, self.sf_name)

    def extra_repr(self):
        return f"nf={self.nf}, nx={self.nx}, {self.sf.describe()}, name={self.sf_name!r}"


def _pair(v):
    return tuple(v) if isinstance(v, (tuple, list)) else (v, v)


def convertible_conv(c: nn.Conv2d):
    if c.groups != 1:
        return False, f"groups={c.groups} (only groups=1 is converted)"
    if c.padding_mode != "zeros":
        return False, f"padding_mode={c.padding_mode!r} (only 'zeros' is converted)"
    if isinstance(c.padding, str):
        return False, f"padding={c.padding!r} (only explicit integer padding is converted)"
    return True, ""


class SFConv2d(nn.Module):
    """``nn.Conv2d`` as unfold (data movement) + SF linear (the reduction)."""

    def __init__(self, conv: nn.Conv2d, name: str, cfg: SFConfig):
        super().__init__()
        ok, why = convertible_conv(conv)
        if not ok:
            raise ValueError(why)
        self.in_channels, self.out_channels = conv.in_channels, conv.out_channels
        self.kernel_size = _pair(conv.kernel_size)
        self.stride, self.padding, self.dilation = _pair(conv.stride), _pair(conv.padding), _pair(conv.dilation)
        self.sf = cfg
        self.sf_name = name
        self.weight = conv.weight
        self.bias = conv.bias
        self.train(conv.training)

    def forward(self, x):
        n, _, h, w = x.shape
        kh, kw = self.kernel_size
        cols = F.unfold(x, (kh, kw), dilation=self.dilation, padding=self.padding, stride=self.stride)
        oh = (h + 2 * self.padding[0] - self.dilation[0] * (kh - 1) - 1) // self.stride[0] + 1
        ow = (w + 2 * self.padding[1] - self.dilation[1] * (kw - 1) - 1) // self.stride[1] + 1
        y = call_linear(cols.transpose(1, 2), self.weight.reshape(self.out_channels, -1), self.bias, self.sf,
                        self.sf_name)
        return y.transpose(1, 2).reshape(n, self.out_channels, oh, ow)

    def extra_repr(self):
        return (f"{self.in_channels}, {self.out_channels}, kernel_size={self.kernel_size}, stride={self.stride}, "
                f"padding={self.padding}, {self.sf.describe()}, name={self.sf_name!r}")


def convertible_norm(norm: nn.LayerNorm):
    from .. import _lib
    if len(norm.normalized_shape) != 1:
        return False, f"normalized_shape={tuple(norm.normalized_shape)} (only the last dimension is converted)"
    if not 1 <= norm.normalized_shape[0] <= _lib.NORM_MOST:
        return False, f"normalized_shape={tuple(norm.normalized_shape)} (1 to {_lib.NORM_MOST} features are converted)"
    for name in ("weight", "bias"):
        if name not in norm._parameters:
            return False, f"its {name} is computed"
        p = norm._parameters[name]
        if p is not None and p.dtype not in _tensor._FLOATS:
            return False, f"its {name} is {p.dtype} (float32, bfloat16 and float16 are converted)"
    return True, ""


class SFLayerNorm(nn.Module):
    """``nn.LayerNorm`` over the last dimension on the B200's own kernel (:func:`layer_norm`); its parameters are the
    source's."""

    def __init__(self, norm: nn.LayerNorm):
        super().__init__()
        ok, why = convertible_norm(norm)
        if not ok:
            raise ValueError(why)
        self.normalized_shape, self.eps = tuple(norm.normalized_shape), norm.eps
        self.weight, self.bias = norm.weight, norm.bias
        self.train(norm.training)

    def forward(self, x):
        if x.shape[-1:] != self.normalized_shape:
            from .._errors import SFShapeError
            raise SFShapeError(f"the input has shape {tuple(x.shape)}, the norm is over {self.normalized_shape[0]} features")
        return _norm.layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.normalized_shape}, eps={self.eps}, weight={self.weight is not None}, bias={self.bias is not None}"


class _Recorded(TorchFunctionMode):
    """The calls of torch functions (operators, methods and attributes of tensors among them) while it is entered."""

    def __init__(self):
        super().__init__()
        self.calls = []                         # (function, arguments, keywords, result)

    def __torch_function__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        self.calls.append((func, args, kwargs or {}, out))
        return out


_PRODUCTS = {torch.mul, torch.multiply, torch.Tensor.mul, torch.Tensor.multiply, torch.Tensor.mul_, torch.Tensor.multiply_}
_RELUS = {F.relu, torch.relu, torch.relu_, torch.Tensor.relu, torch.Tensor.relu_}


def _activation_called(func, args, kwargs):
    """tensor_gated's name for the activation that a recorded call is, or None."""
    options = {k: v for k, v in kwargs.items() if k != "inplace"}
    if func is F.gelu:
        name = {"none": "gelu", "tanh": "gelu_tanh"}.get(options.pop("approximate", "none"))
    else:
        name = "silu" if func is F.silu else "relu" if func in _RELUS else None
    return name if len(args) == 1 and not options else None


def _gate_activation(act):
    """tensor_gated's name for an activation module, known by the one function that it calls; None for any other."""
    t = torch.linspace(-2, 2, 8)
    try:
        with torch.no_grad(), _Recorded() as seen:
            out = act(t)
    except Exception:  # noqa: BLE001  (not an activation, or not one for a vector on the host)
        return None
    if len(seen.calls) != 1:
        return None
    func, args, kwargs, result = seen.calls[0]
    return _activation_called(func, args, kwargs) if args and args[0] is t and result is out else None


def _expression(calls, x, result, projections):
    """What ``result`` is in terms of x by the recorded calls, as text; None where one of them is not a projection, an
    activation or a product of two of these.  ``projections``: their names by (id of the weight, id of the bias)."""
    made = {id(x): "x"}
    for func, args, kwargs, out in calls:
        known = [str(made.get(id(t))) for t in args]
        if func is F.linear and len(args) == 3 and not kwargs:
            made[id(out)] = f"{projections.get((id(args[1]), id(args[2])))}({known[0]})"
        elif func in _PRODUCTS and len(args) == 2 and not kwargs:
            made[id(out)] = " * ".join(sorted(known))
        else:
            act = _activation_called(func, args, kwargs)
            if act is None:
                return None
            made[id(out)] = f"{act}({known[0]})"
    return made.get(id(result))


def _hooked(m):
    """Whether a call of the module does more than its class's forward: by hooks, or a forward set on the module itself."""
    return "forward" in getattr(m, "__dict__", ()) or any(getattr(m, h, None) for h in ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks"))


def gated_block(m: nn.Module):
    """(activation, "") of a gated feed-forward block that :class:`SFGatedFeedForward` can stand for, (None, "") of another
    module, (None, why) of a block that it cannot.  A block is recognised by its children (``gate_proj``, ``up_proj``,
    ``down_proj``, ``act_fn``) and by every call that its forward makes on tensors, in training and in evaluation, with
    gradients and without: three projections, the activation and one product, each of what the ones before have made."""
    parts = [m._modules.get(n) for n in ("gate_proj", "up_proj", "down_proj")]
    if not all(isinstance(p, nn.Linear) for p in parts):
        return None, ""
    gate, up, down = parts
    if any(_custom_forward(p, nn.Linear) for p in parts):
        return None, "a projection has a forward of its own"
    act_fn = getattr(m, "act_fn", None)
    if any(map(_hooked, (m, gate, up, act_fn))):
        return None, "it has hooks"
    act = _gate_activation(act_fn)
    if act is None:
        return None, f"activation {type(act_fn).__name__}"
    if set(m._modules) - {"gate_proj", "up_proj", "down_proj", "act_fn"}:
        return None, "it has other children"
    if m._parameters or m._buffers:
        return None, "it has parameters or buffers of its own"
    if gate.weight.shape != up.weight.shape or gate.weight.dtype != up.weight.dtype:
        return None, "its first two projections differ in shape or type"
    if gate.weight.is_meta:
        return None, "its weights are on the meta device"
    takes = list(inspect.signature(m.forward).parameters.values())
    if len(takes) != 1 or takes[0].kind not in (takes[0].POSITIONAL_ONLY, takes[0].POSITIONAL_OR_KEYWORD):
        return None, "its forward does not take one argument"
    keys = [(id(p.weight), id(p.bias)) for p in parts]
    projections = dict(zip(keys, ("gate", "up", "down")))      # (those that share their parameters share a name)
    g, u, d = map(projections.get, keys)
    want = f"{d}({' * '.join(sorted((f'{act}({g}(x))', f'{u}(x)')))})"
    modes = [(t, t.training) for t in m.modules()]
    try:
        x = torch.linspace(-2, 2, 2 * gate.in_features, device=gate.weight.device).view(2, -1).to(gate.weight.dtype)
        x.requires_grad_()
        grads = (False,) if torch.is_inference_mode_enabled() or gate.weight.is_inference() else (False, True)
        for training in (False, True):
            for t, _ in modes:
                t.training = training
            for grad in grads:
                with torch.set_grad_enabled(grad), _Recorded() as seen:
                    out = m(x)
                # (modes that the forward enters are no calls, but show in what these make)
                if (len(seen.calls) != 5 or _expression(seen.calls, x, out, projections) != want
                        or any(r.requires_grad is not grad or r.dtype is not x.dtype for *_, r in seen.calls)):
                    return None, "it computes something else than down(act(gate(x)) * up(x))"
    except Exception as e:  # noqa: BLE001  (a model's own forward may raise)
        return None, f"its forward did not run on two rows ({type(e).__name__})"
    finally:
        for t, training in modes:
            t.training = training
    return act, ""


class SFGatedFeedForward(nn.Module):
    """A gated feed-forward block ``down(act(gate(x)) * up(x))`` with SF arithmetic on the tensor cores: the first two
    projections and their product are one operator (:func:`tensor_gated`), the last is an SF linear layer.  The
    children and their parameters are the source's."""

    def __init__(self, block: nn.Module, name: str, cfg: SFConfig, down: SFConfig | None = None, *, activation=None):
        """``activation``: what :func:`gated_block` says of the block, where it has been asked."""
        super().__init__()
        if cfg.accumulate != "tensor":
            raise ValueError("a gated block is one operator with accumulate=\"tensor\" only")
        why = ""
        self.activation = activation
        if activation is None:
            self.activation, why = gated_block(block)
        if self.activation is None:
            raise ValueError(why or "not a gated feed-forward block")
        self.sf, self.sf_name = cfg, name
        self.gate_proj, self.up_proj, self.act_fn = block.gate_proj, block.up_proj, block.act_fn
        self.down_proj = SFLinear.from_float(block.down_proj, f"{name}.down_proj" if name else "down_proj", down or cfg)
        self.train(block.training)

    def forward(self, x):
        gate, up = self.gate_proj, self.up_proj
        return self.down_proj(_gated.tensor_gated(x, gate.weight, up.weight, gate.bias, up.bias, activation=self.activation,
                                                  dtype=self.sf.bits, scale=self.sf.scale))

    def extra_repr(self):
        return f"activation={self.activation}, {self.sf.describe()}, name={self.sf_name!r}"


@dataclass
class ConversionReport:
    converted: list = field(default_factory=list)     # (name, kind)
    skipped: list = field(default_factory=list)       # (name, kind, reason)
    shared: list = field(default_factory=list)        # (alias name, converted name)
    kept_sf16: list = field(default_factory=list)     # (name, why)
    attention: str = "float (not converted)"
    widths: dict = field(default_factory=dict)        # name -> bits

    def __repr__(self):
        lines = [f"ConversionReport: {len(self.converted)} converted, {len(self.skipped)} skipped"
                 + (f", {len(self.shared)} shared alias(es)" if self.shared else "")
                 + (f", {len(self.kept_sf16)} kept at sf16" if self.kept_sf16 else "")]
        if self.widths:
            per = {}
            for b in self.widths.values():
                per[b] = per.get(b, 0) + 1
            lines += ["  widths: " + ", ".join(f"sf{b} x {k}" for b, k in sorted(per.items()))]
        lines += [f"  + {n} ({k})" for n, k in self.converted]
        lines += [f"  ^ {n} kept at sf16: {w}" for n, w in self.kept_sf16]
        lines += [f"  attention: {self.attention}"]
        lines += [f"  = {a} is {n} (shared module, converted once)" for a, n in self.shared]
        lines += [f"  - {n} ({k}): {r}" for n, k, r in self.skipped]
        return "\n".join(lines)


def _linear_like(m):
    return isinstance(m, (nn.Linear, SFLinear, SFHFConv1D)) or is_hf_conv1d(m)


def _head_from_output_embeddings(model, linears, embeddings) -> dict:
    get = getattr(model, "get_output_embeddings", None)
    if not callable(get):
        return {}
    try:
        head = get()
    except Exception:  # noqa: BLE001  (a model's own hook may raise)
        return {}
    if isinstance(head, nn.Module) and _linear_like(head):
        return {id(head): "LM head (the model's get_output_embeddings())"}
    return {}


def _heads_tied_to_embeddings(model, linears, embeddings) -> dict:
    def shares(w, e):
        return w is e.weight or (w is not None and w.data_ptr() == e.weight.data_ptr()
                                 and w.numel() == e.weight.numel())
    return {id(m): "LM head (weight tied to the embeddings)" for m in linears
            if any(shares(getattr(m, "weight", None), e) for e in embeddings)}


def _head_by_vocabulary(model, linears, embeddings) -> dict:
    vocab = {e.num_embeddings for e in embeddings}
    hits = [m for m in linears if (getattr(m, "out_features", None) or getattr(m, "nf", None)) in vocab]
    return {id(hits[-1]): "LM head (last layer with the vocabulary's output size)"} if hits else {}


def find_lm_heads(model: nn.Module) -> dict:
    """The LM head(s), {id(module): why}, by the first rule that finds one:
    the model's get_output_embeddings(); a linear tied to an embedding's
    weight; the last linear whose output size is an embedding's vocabulary
    (src/sf/torch/_modules.py:263-292).  The last two need an nn.Embedding."""
    linears = [m for m in model.modules() if _linear_like(m)]
    embeddings = [m for m in model.modules() if isinstance(m, nn.Embedding)]
    for rule in (_head_from_output_embeddings, _heads_tied_to_embeddings, _head_by_vocabulary):
        if rule is not _head_from_output_embeddings and not embeddings:
            return {}
        found = rule(model, linears, embeddings)
        if found:
            return found
    return {}


def _custom_forward(m, base) -> bool:
    return type(m).forward is not base.forward


# layer types with no SF form: reported as skipped, run in float
_NO_SF_FORM = (nn.Conv1d, nn.Conv3d, nn.ConvTranspose1d, nn.ConvTranspose2d, nn.ConvTranspose3d, nn.Bilinear,
               nn.LSTM, nn.GRU, nn.RNN, nn.MultiheadAttention)


def _module_names(model) -> set:
    return {n for n, _ in model.named_modules(remove_duplicate=False)}


def _unknown_names(model, names, what):
    missing = sorted(set(names) - _module_names(model))
    if missing:
        raise ValueError(f"{what}: no module named {', '.join(map(repr, missing))}")


class _Converter:
    """One pass of ``convert``: the width each layer gets, the SF layer that
    replaces it, the report.  A module reached twice (a shared submodule) is
    replaced once and the alias recorded."""

    def __init__(self, cfg, cfg16, per_layer, keep_ids, keep_names, fuse=False):
        self.fuse = fuse                        # gated blocks and layer norms as one operator each
        self.cfg, self.cfg16 = cfg, cfg16
        self.per_layer = per_layer              # path -> SFConfig (widths=)
        self.keep_ids, self.keep_names = keep_ids, keep_names
        self.report = ConversionReport()
        self.replaced = {}                      # id(module) -> (first path, replacement or None)
        self.walked = set()

    def config_for(self, module, path) -> SFConfig:
        if path in self.per_layer:
            c = self.per_layer[path]
        elif self.cfg.bits < 16 and (id(module) in self.keep_ids or path in self.keep_names):
            self.report.kept_sf16.append((path, self.keep_ids.get(id(module)) or "named in keep_sf16"))
            c = self.cfg16
        else:
            c = self.cfg
        self.report.widths[path] = c.bits
        return c

    def _skip(self, path, kind, why):
        self.report.skipped.append((path, kind, why))

    def _make(self, module, path):
        """(SF replacement or None, whether the module is a leaf of the walk)."""
        kind = type(module).__name__
        if self.fuse:
            made = self._fused(module, path, kind)
            if made is not None:
                return made, True
        if isinstance(module, (SFLinear, SFConv2d, SFHFConv1D, SFGatedFeedForward)):
            self.report.converted.append((path, kind + " (already SF)"))
            return None, True
        if isinstance(module, nn.Linear):
            if _custom_forward(module, nn.Linear):
                self._skip(path, kind, f"a subclass of nn.Linear with its own forward ({kind}); runs as it was")
            elif not module.weight.is_floating_point():
                self._skip(path, kind, f"weights stored as {module.weight.dtype}")
            else:
                self.report.converted.append((path, "Linear"))
                return SFLinear.from_float(module, path, self.config_for(module, path)), True
            return None, True
        if is_hf_conv1d(module):
            if not module.weight.is_floating_point():
                self._skip(path, kind, f"weights stored as {module.weight.dtype}")
                return None, True
            self.report.converted.append((path, "Conv1D (Hugging Face)"))
            return SFHFConv1D(module, path, self.config_for(module, path)), True
        if isinstance(module, nn.Conv2d):
            ok, why = convertible_conv(module)
            if not (ok and module.weight.is_floating_point()):
                self._skip(path, "Conv2d", why or f"weights stored as {module.weight.dtype}")
                return None, True
            self.report.converted.append((path, "Conv2d"))
            return SFConv2d(module, path, self.config_for(module, path)), True
        if isinstance(module, _NO_SF_FORM):
            self._skip(path, kind, "no SF version here; runs in float")
            return None, True
        return None, False                      # a container: walk into it

    def _fused(self, module, path, kind):
        """A layer norm's or gated block's replacement, or None: the module is looked at as any other then."""
        if isinstance(module, nn.LayerNorm):
            ok, why = convertible_norm(module)
            if _custom_forward(module, nn.LayerNorm) or "forward" in vars(module):
                self._skip(path, kind, f"a subclass of nn.LayerNorm with its own forward ({kind}); runs as it was")
            elif not ok or _hooked(module):
                self._skip(path, kind, f"{why or 'it has hooks'}; runs as it was")
            else:
                self.report.converted.append((path, "LayerNorm"))
                return SFLayerNorm(module)
            return None
        act, why = gated_block(module)
        at = [f"{path}.{n}" if path else n for n in ("gate_proj", "up_proj", "down_proj")]
        if act and len({self.per_layer.get(p, self.cfg).bits for p in at[:2]}) > 1:
            act, why = None, "its first two projections are given two widths"
        if act is None:
            if why:
                self._skip(path, kind, f"not one operator: {why}; its layers are converted one by one")
            return None
        cfg, _, down = (self.config_for(module._modules[n], p) for n, p in zip(("gate_proj", "up_proj", "down_proj"), at))
        self.report.converted.append((path, "gated feed-forward"))
        return SFGatedFeedForward(module, path, cfg, down, activation=act)

    def replace(self, module, path):
        seen = self.replaced.get(id(module))
        if seen is not None:                    # met before: the same replacement, no second walk
            first, rep = seen
            if rep is not None:
                self.report.shared.append((path, first))
            return rep, True
        rep, leaf = self._make(module, path)
        self.replaced[id(module)] = (path, rep)
        return rep, leaf

    def walk(self, parent, prefix):
        if id(parent) in self.walked:
            return
        self.walked.add(id(parent))
        for name, child in list(parent._modules.items()):
            if child is None:
                continue
            path = f"{prefix}.{name}" if prefix else name
            rep, leaf = self.replace(child, path)
            if rep is not None:
                setattr(parent, name, rep)
            elif not leaf:
                self.walk(child, path)

    def run(self, model):
        rep, leaf = self.replace(model, "")
        if rep is not None:
            model = rep
        elif not leaf:
            self.walk(model, "")
        model._sf_conversion_report = self.report
        return model


class SFPackedLinear(nn.Module):
    """A linear layer whose weight is packed sf codes (buffers ``codes`` int8 and
    ``scale`` float32): an SF layer of accumulate="tensor" laid out once for
    serving.  Its weight does not train; gradients pass to x and the bias."""

    def __init__(self, packed: "_tensor.SFPackedWeight", bias=None, name: str = ""):
        super().__init__()
        self.bits, self.sf_name = packed.bits, name
        self.out_features, self.in_features = packed.shape
        self.register_buffer("codes", packed.codes)
        self.register_buffer("scale", packed.scale)
        self.bias = bias

    def forward(self, x, *, activation=None, residual=None):
        return _tensor.tensor_linear(x, _tensor.SFPackedWeight(self.codes, self.scale, self.bits), self.bias,
                                     activation=activation, residual=residual)

    def _apply(self, fn, recurse=True):
        # .to(dtype), .half() and the like move the layer; its scales stay float32
        scale = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float32:
            self.scale = scale.to(self.scale.device)
        return self

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"dtype=sf{self.bits}, name={self.sf_name!r}")


class SFPackedGatedFeedForward(nn.Module):
    """A :class:`SFGatedFeedForward` laid out once for serving: three packed projections, of which the first two and their
    product are one operator."""

    def __init__(self, gate: SFPackedLinear, up: SFPackedLinear, down: nn.Module, activation: str, name: str = ""):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj = gate, up, down
        self.activation, self.sf_name = activation, name

    def forward(self, x):
        gate, up = (_tensor.SFPackedWeight(p.codes, p.scale, p.bits) for p in (self.gate_proj, self.up_proj))
        return self.down_proj(_gated.tensor_gated(x, gate, up, self.gate_proj.bias, self.up_proj.bias,
                                                  activation=self.activation))

    def extra_repr(self):
        return f"activation={self.activation}, name={self.sf_name!r}"


def pack(model: nn.Module, inplace: bool = False) -> nn.Module:
    """Replace the SF linear layers of accumulate="tensor" (SFLinear, SFHFConv1D)
    by :class:`SFPackedLinear`, and their gated blocks by :class:`SFPackedGatedFeedForward`:
    the weights' codes are made once, and a weight takes one byte an element.  Other
    layers stay as they are; a layer that the model reaches twice is packed once."""
    if not inplace:
        model = copy.deepcopy(model)
    done = {}

    def packed(m):
        if id(m) not in done and isinstance(m, SFGatedFeedForward):
            gate, up = (SFPackedLinear(_tensor.pack_weight(p.weight, m.sf.bits, m.sf.scale), p.bias, f"{m.sf_name}.{n}")
                        for p, n in ((m.gate_proj, "gate_proj"), (m.up_proj, "up_proj")))
            down = packed(m.down_proj) if wanted(m.down_proj) else m.down_proj
            done[id(m)] = (m, SFPackedGatedFeedForward(gate, up, down, m.activation, m.sf_name).train(m.training))
        elif id(m) not in done:
            w = m.weight.t() if isinstance(m, SFHFConv1D) else m.weight
            p = _tensor.pack_weight(w, m.sf.bits, m.sf.scale)
            # (the layer itself is kept, so that its id stays its own)
            done[id(m)] = (m, SFPackedLinear(p, m.bias, m.sf_name).train(m.training))
        return done[id(m)][1]

    def wanted(m):
        return isinstance(m, (SFLinear, SFHFConv1D, SFGatedFeedForward)) and m.sf.accumulate == "tensor"

    if wanted(model):
        return packed(model)
    for parent in list(model.modules()):
        for name, child in list(parent._modules.items()):
            if child is not None and wanted(child):
                setattr(parent, name, packed(child))
    return model


def _keep_plan(model, keep_sf16, bits):
    """(LM heads by id, module names) that stay at sf16 when ``bits`` < 16."""
    if keep_sf16 == "auto":
        return (find_lm_heads(model) if bits < 16 else {}), set()
    if keep_sf16 in (False, None):
        return {}, set()
    if isinstance(keep_sf16, str) or not hasattr(keep_sf16, "__iter__"):
        raise ValueError(f"keep_sf16 must be \"auto\", False or a list of module names, got {keep_sf16!r}")
    names = set(keep_sf16)
    if bits < 16:
        _unknown_names(model, names, "keep_sf16")
    return {}, names


def convert(model: nn.Module, dtype="sf16", scale: str = "per_tensor", headroom: str = "bound",
            inplace: bool = False, *, accumulate: str = "chain", shift=None, calibration: str = "heuristic",
            keep_sf16="auto", attention="auto", nonlinear: str = "float",
            widths: dict | None = None, fuse: bool = False) -> nn.Module:
    """Swap ``nn.Linear``, ``nn.Conv2d`` and Hugging Face ``Conv1D`` for SF
    layers (src/sf/torch/_modules.py:295-537).  ``keep_sf16`` ("auto": the LM
    head; False; or module names) keeps layers at sf16 when ``dtype`` is
    narrower; ``widths`` ({name: dtype}) gives layers their own width.
    ``accumulate="tensor"`` runs the layers on the tensor cores, for a model in
    bfloat16 or float16; it ends at sf8, so "auto" keeps nothing there.  ``fuse`` (with
    accumulate="tensor") also swaps gated feed-forward blocks, whose forward is down(act(gate(x)) *
    up(x)) over children ``gate_proj``, ``up_proj`` and ``down_proj`` and nothing else, and
    ``nn.LayerNorm`` for modules that are one operator each (:class:`SFGatedFeedForward`, :class:`SFLayerNorm`)."""
    if fuse and accumulate != "tensor":
        raise ValueError("fuse=True is for accumulate=\"tensor\"")
    if calibration not in ("heuristic",):
        raise ValueError(f"calibration must be 'heuristic', got {calibration!r}")
    if attention not in ("auto", False, None):
        raise ValueError(f"attention must be \"auto\" or False, got {attention!r}")
    if nonlinear != "float":
        from .._errors import SFUnsupportedError
        raise SFUnsupportedError("nonlinear must be \"float\" here: the integer non-linear ops are not built")
    if accumulate == "wide" and attention == "auto":
        from .._errors import SFUnsupportedError
        raise SFUnsupportedError("accumulate=\"wide\" with attention=\"auto\" runs scaled-dot-product attention "
                                 "on the MX engine, which is not built here; pass attention=False to keep "
                                 "attention in float (the layers still run wide)")
    cfg = SFConfig(_bits_of(dtype), scale, headroom, accumulate, shift)
    if accumulate == "tensor":
        if keep_sf16 not in ("auto", False, None):
            raise ValueError("accumulate=\"tensor\" has no sf16 for keep_sf16 to keep layers at")
        keep_sf16 = False
    if not inplace:
        model = copy.deepcopy(model)
    keep_ids, keep_names = _keep_plan(model, keep_sf16, cfg.bits)
    per_layer = {}
    if widths:
        _unknown_names(model, widths, "widths")
        per_layer = {n: SFConfig(_bits_of(d), scale, headroom, accumulate, shift) for n, d in widths.items()}
    cfg16 = cfg if accumulate == "tensor" else SFConfig(16, scale, headroom, accumulate, shift)
    return _Converter(cfg, cfg16, per_layer, keep_ids, keep_names, fuse).run(model)


def conversion_report(model: nn.Module) -> ConversionReport:
    r = getattr(model, "_sf_conversion_report", None)
    if r is None:
        raise ValueError("model was not produced by sft.convert")
    return r
