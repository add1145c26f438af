"""The AdamW step's refusals and its sf8 rounding rule, without a GPU.

``moment_codes`` restates the rounding of an sf8 moment in NumPy float32,
one IEEE operation at a time as the kernel does it; the GPU tests compare the
kernel's codes with it bit for bit.
"""
import ctypes
from array import array

import numpy as np
import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200 import _lib, build
from superfloat.python_b200._errors import SFShapeError, SFTypeError

BLOCK = 256
f32 = np.float32


def dither(n, seed):
    """Two uniform 16-bit numbers for each element, as float32 in [0, 1)."""
    h = (np.arange(n, dtype=np.uint64) * 0x9E3779B1 + (seed & 0xFFFFFFFF)).astype(np.uint32)
    h ^= h >> np.uint32(16)
    h = (h.astype(np.uint64) * 0x7FEB352D).astype(np.uint32)
    h ^= h >> np.uint32(15)
    h = (h.astype(np.uint64) * 0x846CA68B).astype(np.uint32)
    h ^= h >> np.uint32(16)
    return (h & np.uint32(0xFFFF)).astype(f32) * f32(2.0 ** -16), (h >> np.uint32(16)).astype(f32) * f32(2.0 ** -16)


def levels(c, power):
    c2 = c * c
    return c2 if power == 2 else c2 * c2


def moment_values(codes, scale, power):
    c = codes.astype(f32)
    u = np.repeat(scale * f32(1.0 / 127.0 ** power), BLOCK)[: c.size]
    with np.errstate(invalid="ignore", over="ignore"):
        v = levels(np.abs(c), power) * u
    return np.where(c < 0, -v, v).astype(f32)


def moment_codes(value, u, power):
    """(codes, scales) of float32 moments rounded with the dither ``u``."""
    n = value.size
    pad = np.pad(np.abs(value), (0, -n % BLOCK)).reshape(-1, BLOCK)
    top = pad.max(1)
    top = np.where(top < f32(1e-30), f32(0), top)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(top > 0, f32(127.0 ** power) / top, f32(0)).astype(f32)
        t = (np.abs(value) * np.repeat(inv, BLOCK)[:n]).astype(f32)
    c = np.floor(np.sqrt(t) if power == 2 else np.sqrt(np.sqrt(t))).astype(f32)
    c = np.where(levels(c, power) > t, c - 1, c)
    c = np.where(levels(c + 1, power) <= t, c + 1, c).astype(f32).clip(0, 127)
    low = levels(c, power)
    c = c + ((u * (levels(c + 1, power) - low) < t - low) & (c < 127))
    if power == 4:
        c = np.where((t > 0) & (c == 0), 1, c)
    return np.where(value < 0, -c, c).astype(np.int8), top.astype(f32)


def step_f32(p, g, m, v, step, lr, betas, eps, wd):
    """The moments of one step in float32, one rounding an operation; the parameter in 64 bits."""
    b1, b2 = betas
    m1 = m * f32(b1) + g * f32(1 - b1)
    v1 = v * f32(b2) + (g * f32(1 - b2)) * g
    p1 = p.astype(np.float64) * (1 - lr * wd) - lr / (1 - b1 ** step) * m1.astype(np.float64) / (
        np.sqrt(v1.astype(np.float64)) / np.sqrt(1 - b2 ** step) + eps)
    return p1, m1.astype(f32), v1.astype(f32)


@pytest.mark.parametrize("power", [2, 4])
def test_rounding_keeps_the_value_on_average(power):
    """Over many dithers the mean of the decoded value is the value: the error of a mean of R draws has a
    standard deviation of at most step / (2 sqrt R), step <= (level(127) - level(126)) / level(127) of the scale."""
    rng = np.random.default_rng(1)
    value = (np.abs(rng.standard_normal(BLOCK)) ** (power // 2)).astype(f32)
    if power == 2:
        value *= np.where(rng.random(BLOCK) < 0.5, -1, 1).astype(f32)
    rounds, total = 2000, np.zeros(BLOCK)
    seen = np.zeros(BLOCK, bool)
    for r in range(rounds):
        code, top = moment_codes(value, dither(BLOCK, 7919 * r)[0], power)
        total += moment_values(code, top, power)
        seen |= np.abs(code) == 1
    c = np.floor((np.abs(value) / top[0]) ** (1 / power) * 127)
    step = (levels(c + 1, power) - levels(c, power)) / 127.0 ** power * top[0]
    off = np.abs(total / rounds - value)
    kept = ~seen | (power == 2)                       # a second moment below its first level is held at it
    assert (off[kept] <= 5 * step[kept] / (2 * np.sqrt(rounds)) + 2.0 ** -20 * np.abs(value[kept])).all()


@pytest.mark.parametrize("power", [2, 4])
def test_rounding_takes_a_neighbouring_level(power):
    rng = np.random.default_rng(2)
    value = (rng.standard_normal(1000) ** (power // 2 * 3)).astype(f32)
    if power == 4:
        value = np.abs(value)
    code, top = moment_codes(value, dither(1000, 3)[1], power)
    c = np.abs(code).astype(np.float64)
    t = np.abs(value).astype(np.float64) / np.repeat(top, BLOCK)[:1000] * 127.0 ** power
    slack = 1e-5 * (t + 1)
    assert ((c + 1) ** power >= t - slack).all()
    assert (((c - 1).clip(0) ** power <= t + slack) | (c <= 1)).all()
    assert (np.sign(code) * np.sign(value) >= 0).all()


def test_zero_and_tiny_blocks():
    value = np.zeros(600, f32)
    value[256:512] = f32(1e-31)
    value[512] = f32(2.0)
    code, top = moment_codes(value, dither(600, 0)[0], 2)
    assert (code[:512] == 0).all() and top[0] == 0 and top[1] == 0
    assert code[512] == 127 and top[2] == 2.0 and (moment_values(code, top, 2)[512] == f32(2.0))


def _cpu(n=8, dtype=torch.float32):
    return torch.zeros(n, dtype=dtype)


def test_refusals():
    p, g, m, v = _cpu(), _cpu(), _cpu(), _cpu()
    ok = dict(step=1, lr=1e-3)
    with pytest.raises(SFShapeError, match="CUDA device"):
        sft.adamw_step([p], [g], [m], [v], **ok)
    with pytest.raises(SFShapeError, match="2 gradients"):
        sft.adamw_step([p], [g, g], [m], [v], **ok)
    with pytest.raises(SFTypeError, match="float64"):
        sft.adamw_step([p.double()], [g.double()], [m], [v], **ok)
    with pytest.raises(SFTypeError, match="its gradient"):
        sft.adamw_step([p], [g.half()], [m], [v], **ok)
    for bad in (0, -1, 1.5, True):
        with pytest.raises(ValueError, match="step"):
            sft.adamw_step([p], [g], [m], [v], step=bad, lr=1e-3)
    for kw in (dict(lr=-1.0), dict(lr=float("nan")), dict(lr=1.0, eps=-1e-8), dict(lr=1.0, weight_decay=float("inf")),
               dict(lr=1.0, betas=(1.0, 0.9)), dict(lr=1.0, betas=(0.9,))):
        with pytest.raises(ValueError):
            sft.adamw_step([p], [g], [m], [v], step=1, **kw)
    with pytest.raises(SFTypeError, match="lr"):
        sft.adamw_step([p], [g], [m], [v], step=1, lr=torch.tensor(1e-3))
    with pytest.raises(ValueError, match="kind"):
        sft.moment_values([m], "third")
    with pytest.raises(ValueError, match="state"):
        sft.AdamW([torch.nn.Parameter(p)], state="sf4")
    opt = sft.AdamW([torch.nn.Parameter(p)])
    opt.param_groups[0]["params"][0].grad = g
    with pytest.raises(SFTypeError, match="CUDA"):
        opt.step()
    sft.adamw_step([], [], [], [], **ok)              # nothing to do


def test_dense_rule():
    from superfloat.python_b200.torch._optim import _dense
    t = torch.zeros(4, 6)
    assert _dense(t) and _dense(t.t()) and _dense(torch.zeros(0)) and _dense(torch.zeros(3, 1, 2).transpose(0, 1))
    assert not _dense(t[:, :5]) and not _dense(t[0].expand(3, 6)) and not _dense(t[::2])


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _call(lib, rows, dtype=0, sf8=0, step=1):
    words = array("q", [w for r in rows for w in r])
    return lib.sfb_adamw(words.buffer_info()[0], len(rows), dtype, sf8, 1e-3, 0.9, 0.999, 1e-8, 0.0, step, 0, None, None)


def test_the_library_refuses_before_it_launches(lib):
    """Addresses that no launch ever sees: each table is refused on the host."""
    a = 1 << 20
    good = [a, 2 * a, 3 * a, 4 * a, 0, 0, 1000, 0]
    assert _call(lib, [good], dtype=1) == _lib.SFB_EINVAL and b"element type" in lib.sfb_last_error()
    assert _call(lib, [good], step=0) == _lib.SFB_EINVAL
    assert _call(lib, [[0] + good[1:]]) == _lib.SFB_EINVAL and b"null" in lib.sfb_last_error()
    assert _call(lib, [[a + 2] + good[1:]]) == _lib.SFB_EINVAL and b"aligned" in lib.sfb_last_error()
    assert _call(lib, [good[:6] + [-1, 0]]) == _lib.SFB_EINVAL
    assert _call(lib, [good], sf8=1) == _lib.SFB_EINVAL              # no scales
    assert _call(lib, [good, good]) == _lib.SFB_EINVAL and b"given twice" in lib.sfb_last_error()
    shifted = [5 * a, 6 * a, 7 * a, 8 * a, 0, 0, 1000, 0]
    for word in range(4):                                            # one tensor's end in another's start
        other = list(shifted)
        other[word] = a + 3996
        assert _call(lib, [good, other]) == _lib.SFB_EINVAL, word
    assert _call(lib, [good[:1] + [a] + good[2:]]) == _lib.SFB_EINVAL
    assert lib.sfb_adamw(None, 1, 0, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 0, None, None) == _lib.SFB_EINVAL
    assert lib.sfb_adamw(None, 0, 0, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 0, None, None) == _lib.SFB_OK
    assert lib.sfb_sf8_values(None, 0, 3, None) == _lib.SFB_EINVAL
    assert lib.sfb_adamw_advance(None, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, None) == _lib.SFB_EINVAL
    assert ctypes.sizeof(ctypes.c_int64) * _lib.ADAMW_WORDS == 64
