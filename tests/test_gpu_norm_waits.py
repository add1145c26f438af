"""Waits of a long row's norm that run out while a cluster has rows left to do: what is lost is NaN, all of the rest is as
ever, the call ends and is counted."""
import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200 import _lib
from test_gpu_norm import randn

pytestmark = pytest.mark.gpu
# more rows than clusters fit the GPU: two, four and eight CTAs to a row, rows that do not start on 16 bytes
SIZES = [(600, 8200), (600, 8201), (300, 32768), (200, 65536)]


def step(x, w, dy):
    x = x.detach().requires_grad_()
    y = sft.layer_norm(x, w, w)
    return y.detach(), torch.autograd.grad(y, x, dy)[0]


def limited(polls, stall, fn, *args):
    _lib.load().sfb_wide_wait_limit(polls, stall)
    try:
        return fn(*args)
    finally:
        _lib.load().sfb_wide_wait_limit(0, 0)


def backward_on_this_thread(x, w, dy):
    """(The limit is the calling thread's: the backward pass by the library's call, as the graph's thread makes it.)"""
    from superfloat.python_b200.torch import _norm

    class Ctx:
        pass

    _, rows, stats = _norm._forward(x, w, w, 1e-5, True)
    ctx = Ctx()
    ctx.saved_tensors = rows, w, stats
    ctx.call = (*rows.shape, x.dtype, w.dtype, w.dtype, x.device, x.shape)
    ctx.needs_input_grad = (True, False, False, False)
    return lambda: _norm._gradients(ctx, dy)[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,d", SIZES)
def test_parts_that_never_come(gpu, m, d, dtype):
    x, w, dy = randn(m, d, dtype=dtype), randn(d, seed=1, dtype=dtype), randn(m, d, seed=2, dtype=dtype)
    want = step(x, w, dy)
    before = sft.tensor_failures()
    assert bool(limited(2000, 1, sft.layer_norm, x, w, w).isnan().all())
    assert bool(limited(2000, 1, backward_on_this_thread(x, w, dy)).isnan().all())
    assert sft.tensor_failures() >= before + 2
    again = step(x, w, dy)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("m,d", SIZES)
def test_waits_of_one_poll(gpu, m, d):
    """Some waits run out and some do not, in any warp and row: each element is right or NaN."""
    x, w, dy = randn(m, d, dtype=torch.bfloat16), randn(d, seed=1), randn(m, d, seed=2, dtype=torch.bfloat16)
    want = step(x, w, dy)
    for _ in range(3):
        before = sft.tensor_failures()
        y = limited(1, 0, sft.layer_norm, x, w, w)
        g = limited(1, 0, backward_on_this_thread(x, w, dy))
        assert bool((y.isnan() | (y == want[0])).all()) and bool((g.isnan() | (g == want[1])).all())
        assert not bool(y.isnan().any() | g.isnan().any()) or sft.tensor_failures() > before
    again = step(x, w, dy)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
