"""The dither of sf8 moments: another one each step, unless the caller gives it."""
import numpy as np
import pytest


import superfloat.python_b200.torch as sft
from superfloat.python_b200.torch import _optim
from test_adamw_host import BLOCK, dither, f32, moment_codes, moment_values


def test_the_step_is_the_default(monkeypatch):
    seen = []
    monkeypatch.setattr(_optim, "_launch", lambda *a: seen.append(a[6]))
    for step in (1, 2, 3):
        sft.adamw_step([], [], [], [], step=step, lr=1e-3)
        sft.adamw_step([], [], [], [], step=step, lr=1e-3, dither=0)
    assert seen == [1, 0, 2, 0, 3, 0]


@pytest.mark.parametrize("fixed", [False, True])
def test_why_it_has_to_change(fixed):
    """A second moment without gradients decays by 0.999 a step, less than a code's step of 1 - (126 / 127)^4 = 3.1 %:
    over 400 steps to 0.670 of itself.  The draws are independent from step to step, each off by at most half of
    3.1 % and unbiased, so the mean of 256 has a standard deviation of sqrt(400) x 1.6 % / 16 = 2 % at most.  With one
    dither for all steps most elements stay where they are."""
    codes, scale = np.full(BLOCK, 100, np.int8), np.ones(1, f32)
    codes[0] = 127                                     # holds the block's scale; it decays as the scale does
    first = moment_values(codes, scale, 4)
    for step in range(1, 401):
        v = moment_values(codes, scale, 4) * f32(0.999)
        v[0] = f32(1.0)
        codes, scale = moment_codes(v, dither(BLOCK, 7 if fixed else step)[1], 4)
    left = moment_values(codes, scale, 4)[1:] / first[1:]
    if fixed:
        assert (left == 1).mean() > 0.9
    else:
        assert abs(float(left.mean()) - 0.999 ** 400) < 4 * 0.02


