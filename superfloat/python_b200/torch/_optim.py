"""AdamW over many tensors at once, with moments in float32 or in sf8.

The straight-through training of converted layers (``sf::linear`` and its
kin) keeps float parameters; this is the optimizer step that goes with it.
The reference trains with torch's optimizers and has no counterpart.

    p <- p (1 - lr wd) - lr / bc1 * m / (sqrt(v / bc2) + eps)
    m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2,   bc_i = 1 - b_i^step

An sf8 moment is int8 codes in [-127, 127] with one float32 scale for every
256 elements in storage order; a code c stands for ``scale (c / 127)^2`` with
c's sign in the first moment and ``scale (c / 127)^4`` in the second.  Codes
are rounded by a dither that keeps the value unbiased.  ``csrc/sfb_adamw.cu``
has the kernels and the reasons.
"""
from __future__ import annotations

import math
from array import array
from dataclasses import dataclass

import torch

from .. import _lib
from .._errors import SFShapeError, SFTypeError, SFUnsupportedError

BLOCK = 256                        # elements that share a scale
SF8_FROM = 4096                    # AdamW(state="sf8") keeps smaller tensors' moments in float32
_ELEMENT = {torch.float32: _lib.ELEMENT["float32"], torch.bfloat16: _lib.ELEMENT["bfloat16"],
            torch.float16: _lib.ELEMENT["float16"]}
_POWER = {"first": 2, "second": 4}
# Between the dithers of neighbouring tensors.  All draw from one sequence (csrc/sfb_adamw.cu, `mixed`), each from its
# own place: element e of tensor i + 1 draws what element e + 1 of tensor i draws eight steps later.  Each draw is
# uniform, so each moment's rounding is unbiased; draws of different tensors are not independent over steps.
_SEED_STEP = 0x9E3779B9


@dataclass
class SF8Moment:
    """A moment of ``codes.numel()`` elements: int8 codes in the parameter's
    storage order, and a float32 scale for every 256 of them."""

    codes: torch.Tensor
    scale: torch.Tensor

    @classmethod
    def zeros(cls, n: int, device) -> "SF8Moment":
        return cls(torch.zeros(n, dtype=torch.int8, device=device),
                   torch.zeros(-(-n // BLOCK), dtype=torch.float32, device=device))


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one stretch of memory, each place once."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _check_sf8(m: SF8Moment, n: int, device, what: str, i: int) -> None:
    c, s = m.codes, m.scale
    if c.dtype != torch.int8 or s.dtype != torch.float32:
        raise SFTypeError(f"{what} {i}: an sf8 moment has int8 codes and float32 scales, got {c.dtype} and {s.dtype}")
    if c.numel() != n or s.numel() != -(-n // BLOCK):
        raise SFShapeError(f"{what} {i}: {n} elements need {n} codes and {-(-n // BLOCK)} scales, got {c.numel()} and "
                           f"{s.numel()}")
    if c.device != device or s.device != device:
        raise SFShapeError(f"{what} {i}: the moment is not on {device}")
    if not (c.is_contiguous() and s.is_contiguous()):
        raise SFShapeError(f"{what} {i}: codes and scales must be contiguous")
    if n and c.data_ptr() % 4:
        raise SFShapeError(f"{what} {i}: the codes must start on a 4-byte boundary")


def _check_rates(lr, betas, eps, weight_decay):
    for name, v in (("lr", lr), ("eps", eps), ("weight_decay", weight_decay)):
        if isinstance(v, torch.Tensor):
            raise SFTypeError(f"{name} must be a number, not a tensor")
        if not (v >= 0 and math.isfinite(v)):
            raise ValueError(f"{name} must be a finite number of at least 0, got {v!r}")
    if len(betas) != 2 or not all(0 <= b < 1 for b in betas):
        raise ValueError(f"betas must be two numbers in [0, 1), got {betas!r}")


def _buckets(params, grads, exp_avg, exp_avg_sq):
    """{(device index, element type, sf8): [table words]}, one entry for each
    tensor, after the checks; and the gradients that had to be laid out."""
    buckets, kept, seen = {}, [], set()
    for i, (p, g, m, v) in enumerate(zip(params, grads, exp_avg, exp_avg_sq)):
        dt, shape, device = _ELEMENT.get(p.dtype), p.shape, p.device
        if dt is None:
            raise SFTypeError(f"adamw: tensor {i} is {p.dtype}; float32, bfloat16 and float16 are supported")
        if g.dtype != p.dtype:
            raise SFTypeError(f"adamw: tensor {i} is {p.dtype} and its gradient {g.dtype}")
        if not p.is_cuda or g.device != device:
            raise SFShapeError(f"adamw: tensor {i} and its gradient must be on one CUDA device, got {device} and "
                               f"{g.device}")
        if g.layout != torch.strided:
            raise SFUnsupportedError(f"adamw: tensor {i} has a gradient that is not strided")
        if g.shape != shape:
            raise SFShapeError(f"adamw: tensor {i} has shape {tuple(shape)}, its gradient {tuple(g.shape)}")
        plain = p.is_contiguous()
        if not plain and not _dense(p):
            raise SFShapeError(f"adamw: tensor {i} has gaps or overlaps in memory (shape {tuple(shape)}, strides "
                               f"{p.stride()})")
        if not (g.is_contiguous() if plain else g.stride() == p.stride()):
            with torch.no_grad():
                g = torch.empty_strided(shape, p.stride(), dtype=g.dtype, device=device).copy_(g)
            kept.append(g)
        n = p.numel()
        at = p.data_ptr()
        if n and at in seen:                           # (overlaps within a launch are the library's to find)
            raise SFShapeError(f"adamw: tensor {i} is given twice")
        seen.add(at)
        sf8 = isinstance(m, SF8Moment)
        if sf8 != isinstance(v, SF8Moment):
            raise SFTypeError(f"adamw: tensor {i} has one moment in sf8 and one that is not")
        if sf8:
            _check_sf8(m, n, device, "adamw: first moment of tensor", i)
            _check_sf8(v, n, device, "adamw: second moment of tensor", i)
            words = (at, g.data_ptr(), m.codes.data_ptr(), v.codes.data_ptr(), m.scale.data_ptr(),
                     v.scale.data_ptr(), n, (i * _SEED_STEP) & 0xFFFFFFFF)
        else:
            for t in (m, v):
                if t.dtype != torch.float32:
                    raise SFTypeError(f"adamw: tensor {i} has a moment of {t.dtype}; float32 or SF8Moment")
                if t.device != device or t.shape != shape or not (t.is_contiguous() if plain else t.stride() == p.stride()):
                    raise SFShapeError(f"adamw: tensor {i} has a moment of another shape, layout or device")
            words = (at, g.data_ptr(), m.data_ptr(), v.data_ptr(), 0, 0, n, 0)
        key = (p.get_device(), dt, sf8)
        if key not in buckets:
            buckets[key] = array("q")
        buckets[key].extend(words)
    return buckets, kept


def _check_launches(launches) -> None:
    """What the library refuses of each (key, table), before any of them is launched: a step
    happens as a whole or not at all."""
    for (_, dt, sf8), words in launches:
        _lib.adamw_check(words.buffer_info()[0], len(words) // _lib.ADAMW_WORDS, dt, sf8)


def _launch(buckets, lr, betas, eps, weight_decay, step, dither, constants=None):
    for (index, dt, sf8), words in buckets.items():
        with _lib.on_device(index) as d:
            _lib.adamw(words.buffer_info()[0], len(words) // _lib.ADAMW_WORDS, dt, sf8, float(lr),
                       (float(betas[0]), float(betas[1])), float(eps), float(weight_decay), int(step),
                       dither & 0xFFFFFFFF, constants, d.stream)


def _changed(params):
    """Counts the step in the parameters' versions: what autograd saved of them,
    and the codes that a chain or wide layer keeps for its weight, are of before."""
    torch.autograd.graph.increment_version([p for p in params if not p.is_inference()])


def adamw_step(params, grads, exp_avg, exp_avg_sq, *, step: int, lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.0, dither: int | None = None) -> None:
    """One AdamW step on lists of CUDA tensors, in place, on each device's
    current stream.

    ``params`` and ``grads``: float32, bfloat16 or float16 tensors without gaps
    in memory (a gradient of another layout is copied).  ``exp_avg`` and
    ``exp_avg_sq``: float32 tensors of the parameter's layout, or
    :class:`SF8Moment`; both of a parameter's moments are of one kind.  ``step``
    counts from 1.  ``dither`` seeds the rounding of sf8 moments and is another number
    each step, the step itself if it is not given: rounded the same way each time, a
    moment that changes by less than a code's step would never move.  The arithmetic is float32; a 16-bit parameter
    is rounded to nearest once.  A parameter that is given twice is refused, and so
    is a tensor that overlaps another which the same launch (one for each device,
    type and kind of moments) writes.  Nothing of a refused call has run."""
    if not len(params) == len(grads) == len(exp_avg) == len(exp_avg_sq):
        raise SFShapeError(f"adamw: {len(params)} parameters, {len(grads)} gradients, {len(exp_avg)} and "
                           f"{len(exp_avg_sq)} moments")
    if isinstance(step, bool) or not isinstance(step, int) or step < 1:
        raise ValueError(f"step must be an int of at least 1, got {step!r}")
    _check_rates(lr, betas, eps, weight_decay)
    buckets, _kept = _buckets(params, grads, exp_avg, exp_avg_sq)
    _check_launches(list(buckets.items())[1:])         # (the first one's own call checks it)
    _launch(buckets, lr, betas, eps, weight_decay, step, step if dither is None else dither)
    _changed(params)


def moment_values(moments, kind: str) -> list:
    """The float32 values of moments: what the codes of each
    :class:`SF8Moment` stand for, flat in storage order, and float32 moments as
    they are.  ``kind``: "first" or "second"."""
    if kind not in _POWER:
        raise ValueError(f"kind must be \"first\" or \"second\", got {kind!r}")
    out, tables = [], {}
    for i, m in enumerate(moments):
        if not isinstance(m, SF8Moment):
            out.append(m)
            continue
        n = m.codes.numel()
        if not m.codes.is_cuda:
            raise SFShapeError(f"moment {i} must be on a CUDA device, got {m.codes.device}")
        _check_sf8(m, n, m.codes.device, "moment", i)
        out.append(torch.empty(n, dtype=torch.float32, device=m.codes.device))
        tables.setdefault(m.codes.get_device(), array("q")).extend(
            (out[-1].data_ptr(), m.codes.data_ptr(), 0, 0, m.scale.data_ptr(), 0, n, 0))
    for index, words in tables.items():
        with _lib.on_device(index) as d:
            _lib.sf8_values(words.buffer_info()[0], len(words) // _lib.ADAMW_WORDS, _POWER[kind], d.stream)
    return out


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is one launch for the tensors of each type.

    ``state``: "float32", or "sf8" for moments of one byte an element (tensors
    below 4096 elements, biases and norms mostly, keep float32 moments).
    ``dither_seed`` moves the rounding of sf8 moments on by so many steps: two runs
    draw apart from each other where their seeds differ by more than their steps.
    The parameters of each group draw as those of the first.
    ``capturable=True`` keeps the step count on the device, so that ``step()``
    can be captured into a CUDA graph and replayed; the other settings are
    then those of the capture.  Every parameter needs its gradient then.  A
    replay changes the parameters without their versions telling: clear the codes
    that chain and wide layers keep (``sft.weight_cache.clear()``,
    ``sft.wide_weight_cache.clear()``) before one runs outside the graph.

    >>> opt = sft.AdamW(model.parameters(), lr=1e-4, state="sf8")
    >>> loss.backward(); opt.step(); opt.zero_grad()
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, *,
                 state: str = "float32", dither_seed: int = 0, capturable: bool = False):
        _check_rates(lr, betas, eps, weight_decay)
        if state not in ("float32", "sf8"):
            raise ValueError(f"state must be \"float32\" or \"sf8\", got {state!r}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state=state,
                                      dither_seed=int(dither_seed), capturable=bool(capturable)))

    @staticmethod
    def _check_param(p):
        if _ELEMENT.get(p.dtype) is None or not p.is_cuda:
            raise SFTypeError(f"AdamW: a parameter of {p.dtype} on {p.device}; float32, bfloat16 and float16 on a "
                              f"CUDA device are supported")

    def _begin(self, p, group):
        st = self.state[p]
        if st:
            return st
        if group["state"] == "sf8" and p.numel() >= SF8_FROM:
            m, v = SF8Moment.zeros(p.numel(), p.device), SF8Moment.zeros(p.numel(), p.device)
            st["exp_avg"], st["exp_avg_scale"] = m.codes, m.scale
            st["exp_avg_sq"], st["exp_avg_sq_scale"] = v.codes, v.scale
        else:
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        st["step"] = 0
        return st

    @staticmethod
    def _moments(st):
        if "exp_avg_scale" in st:
            return (SF8Moment(st["exp_avg"], st["exp_avg_scale"]),
                    SF8Moment(st["exp_avg_sq"], st["exp_avg_sq_scale"]))
        return st["exp_avg"], st["exp_avg_sq"]

    def _counter(self, group):
        """The group's step counter and constants on the device (capturable)."""
        c = group.get("_counter")
        device = group["params"][0].device
        if c is None or c[0].device != device:
            if torch.cuda.is_current_stream_capturing():
                raise SFUnsupportedError("AdamW: take one step before the capture, so that the moments and the step "
                                         "counter exist")
            done = max((self.state[p].get("step", 0) for p in group["params"] if p in self.state), default=0)
            c = (torch.full((1,), done, dtype=torch.int64, device=device),
                 torch.zeros(_lib.ADAMW_CONSTANTS, dtype=torch.uint8, device=device))
            group["_counter"] = c
        return c

    def _count_on_host(self, group):
        """The device's step count into the parameters' states, where the group was capturable."""
        if group.get("_counter") is not None:
            done = int(group["_counter"][0])
            for p in group["params"]:
                if self.state.get(p):
                    self.state[p]["step"] = done
            group["_counter"] = None

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        todo = []                                      # everything is checked before anything runs
        for group in self.param_groups:
            _check_rates(group["lr"], group["betas"], group["eps"], group["weight_decay"])
            with_grad = [p for p in group["params"] if p.grad is not None]
            if not with_grad:
                continue
            for p in with_grad:
                self._check_param(p)
            capturing = torch.cuda.is_current_stream_capturing()
            if capturing and not group["capturable"]:
                raise SFUnsupportedError("AdamW: a captured step needs capturable=True (the step count is on the "
                                         "host otherwise, and every replay would repeat it)")
            if capturing and any(not self.state.get(p) for p in with_grad):
                raise SFUnsupportedError("AdamW: take one step before the capture, so that the moments and the step "
                                         "counter exist")
            if not group["capturable"]:
                self._count_on_host(group)
            todo += (self._device_step if group["capturable"] else self._host_steps)(group, with_grad)
        launches = [item for _, buckets, *_ in todo for item in buckets.items()]
        _check_launches(launches[0 if todo and todo[0][3] is None else 1:])
        for group, buckets, params, step, _kept in todo:
            rates = group["lr"], group["betas"], group["eps"], group["weight_decay"]
            if step is None:
                counter, constants = group["_counter"]
                with _lib.on_device(counter.get_device()) as d:
                    _lib.adamw_advance(counter.data_ptr(), constants.data_ptr(), float(rates[0]),
                                       tuple(map(float, rates[1])), float(rates[2]), float(rates[3]),
                                       group["dither_seed"] & 0xFFFFFFFF, d.stream)
                _launch(buckets, *rates, 1, 0, constants.data_ptr())
            else:
                _launch(buckets, *rates, step, group["dither_seed"] + step)
                for p in params:
                    self.state[p]["step"] = step
            _changed(params)
        return loss

    def _tables(self, params):
        moments = [self._moments(self.state[p]) for p in params]
        return _buckets(params, [p.grad for p in params], [m for m, _ in moments], [v for _, v in moments])

    def _host_steps(self, group, with_grad):
        """[(group, tables, parameters, their step, gradients laid out)], one for each step count in the group."""
        by_step = {}
        for p in with_grad:
            by_step.setdefault(self._begin(p, group)["step"] + 1, []).append(p)
        steps = []
        for step, params in by_step.items():
            buckets, kept = self._tables(params)
            steps.append((group, buckets, params, step, kept))
        return steps

    def _device_step(self, group, with_grad):
        """The same for a group whose step count is on the device (the step is None)."""
        if len(with_grad) != len(group["params"]):
            raise SFUnsupportedError("AdamW: with capturable=True every parameter of the group needs its gradient "
                                     "(one step count serves the group)")
        if len({p.device for p in with_grad}) != 1:
            raise SFUnsupportedError("AdamW: with capturable=True a group's parameters are on one device")
        for p in with_grad:
            self._begin(p, group)
        self._counter(group)
        buckets, kept = self._tables(with_grad)
        return [(group, buckets, with_grad, None, kept)]

    def moments(self, p) -> tuple:
        """The float32 values of a parameter's two moments, in its shape."""
        st = self.state.get(p)
        if not st:
            raise ValueError("the parameter has not been stepped yet")
        m, v = self._moments(st)
        if isinstance(m, SF8Moment):
            m, v = moment_values([m], "first")[0], moment_values([v], "second")[0]
            m, v = (torch.as_strided(t, p.shape, p.stride()) for t in (m, v))
        return m, v

    def steps_done(self, p) -> int:
        """How many steps the parameter has taken (reads the device with capturable=True)."""
        for group in self.param_groups:
            if any(q is p for q in group["params"]) and group.get("_counter") is not None:
                return int(group["_counter"][0])
        return self.state[p]["step"] if self.state.get(p) else 0

    def state_dict(self):
        """As torch's; a group's device counter is saved as its step count."""
        for group in self.param_groups:
            if group.get("_counter") is not None:
                done = int(group["_counter"][0])
                for p in group["params"]:
                    if self.state.get(p):
                        self.state[p]["step"] = done
        d = super().state_dict()
        for g in d["param_groups"]:
            g.pop("_counter", None)
        return d

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As torch's, but the moments keep their own types (torch would cast them to the
        parameter's), and values go into the buffers that the optimizer has where they
        fit: a captured step names those, and goes on from what was loaded.  sf8 moments
        are in storage order: the parameters' strides are those of the saved run."""
        groups = state_dict["param_groups"]
        old, counters = dict(self.state), [g.get("_counter") for g in self.param_groups]
        super().load_state_dict({**state_dict, "state": {}})
        saved = iter([i for g in groups for i in g["params"]])
        self.state.clear()
        for g, counter in zip(self.param_groups, counters):
            for p in g["params"]:
                st, mine = state_dict["state"].get(next(saved)), old.get(p)
                if not st and mine and counter is not None:
                    st = {k: torch.zeros_like(t) if isinstance(t, torch.Tensor) else 0 for k, t in mine.items()}
                if st:
                    self.state[p] = {k: self._loaded(p, t, (mine or {}).get(k)) if isinstance(t, torch.Tensor) else t
                                     for k, t in st.items()}
            if counter is not None:
                counter[0].fill_(max((self.state[p]["step"] for p in g["params"] if self.state.get(p)), default=0))
            g["_counter"] = counter if g["capturable"] else None

    @staticmethod
    def _loaded(p, t, mine):
        """The values of a saved tensor in the parameter's own (``mine``) or, where they do not fit, a new one."""
        if mine is None or mine.is_inference() or (mine.shape, mine.dtype, mine.device) != (t.shape, t.dtype, p.device):
            if t.shape == p.shape and t.dtype == torch.float32:
                mine = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            else:
                mine = torch.empty_like(t, device=p.device)
        return mine.copy_(t)
