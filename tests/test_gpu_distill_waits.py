"""Waits of the distillation loss that run out while a cluster has rows left to do: what is lost is NaN, all of the rest is as
ever, the call ends and is counted."""
import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200 import _lib
from test_gpu_distill import entries, randn

pytestmark = pytest.mark.gpu
# rows, vocabulary, entries, more rows than clusters fit the GPU: a CTA to a row, one whose entries take longer than its row,
# clusters of 2 and of 8, parts that shared memory does not hold
SIZES = [(2000, 9000, 3), (3000, 33, 1024), (1500, 20000, 64), (300, 120001, 5)]


def step(x, t, i, w, reduction="mean"):
    z = x.detach().requires_grad_()
    loss = sft.distill_loss(z, t, i, row_weight=w, reduction=reduction)
    return loss.detach(), torch.autograd.grad(loss, z, torch.ones_like(loss))[0]


def limited(polls, stall, *args):
    _lib.load().sfb_wide_wait_limit(polls, stall)
    try:
        return step(*args)
    finally:
        _lib.load().sfb_wide_wait_limit(0, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,v,k", SIZES)
def test_parts_that_never_come(gpu, m, v, k, dtype):
    """Every cluster gives up at its first row: all rows that count are NaN, the others 0."""
    x, (t, i) = randn(m, v, dtype=dtype), entries(m, v, k, absent=False)
    w = torch.arange(m, device="cuda") % 7 != 3
    want = step(x, t, i, w)
    assert not bool(want[0].isnan()) and not bool(want[1].isnan().any())
    before = sft.tensor_failures()
    for reduction in ("mean", "sum", "none"):
        loss, g = limited(2000, 1, x, t, i, w, reduction)
        if reduction == "none":
            assert torch.equal(loss.isnan(), w) and not bool(loss[~w].any())
        else:
            assert bool(loss.isnan())
        assert bool(g[w].isnan().all()) and not bool(g[~w].any())
    assert sft.tensor_failures() >= before + 3
    again = step(x, t, i, w)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("m,v,k", SIZES)
def test_waits_of_one_poll(gpu, m, v, k):
    """Some waits run out and some do not, in any warp and row: each row's loss and each element is right or NaN."""
    x, (t, i) = randn(m, v, dtype=torch.bfloat16), entries(m, v, k, absent=False)
    w = torch.arange(m, device="cuda") % 7 != 3
    want = step(x, t, i, w)
    rows = step(x, t, i, w, "none")
    before = sft.tensor_failures()
    for _ in range(3):
        loss, g = limited(1, 0, x, t, i, w)
        assert bool(loss.isnan()) or torch.equal(loss, want[0])
        assert bool((g.isnan() | (g == want[1])).all()) and not bool(g[~w].any())
        loss, g = limited(1, 0, x, t, i, w, "none")
        assert bool((loss.isnan() | (loss == rows[0])).all()) and not bool(loss[~w].any())
        lost = loss.isnan()
        assert bool(g[lost].isnan().all()) and torch.equal(g[~lost], rows[1][~lost])
        assert not bool(lost.any()) or sft.tensor_failures() > before
    again = step(x, t, i, w)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
