"""Gradients of the distillation loss whose rows lie on 16 bytes otherwise than the logits': each thread's part of a row is
what other threads have brought in."""
import pytest
import torch

import superfloat.python_b200.torch as sft
from test_gpu_distill import TYPES, check, entries, randn

pytestmark = pytest.mark.gpu


def laid_out(x, stride):
    """x with rows that start on 16 bytes, `stride` apart."""
    return torch.zeros(x.shape[0], stride, dtype=x.dtype, device="cuda")[:, :x.shape[1]].copy_(x)


# rows and vocabulary: parts shorter than a warp's vectors, many rows of one cluster after another, parts that shared memory
# does not hold
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,v", [(5, 1), (3000, 33), (3000, 250), (2000, 5001), (300, 50257), (5, 120001)])
def test_a_compact_gradient_is_the_aligned_one(gpu, m, v, dtype):
    """The logits' rows start on 16 bytes in both layouts, so that the sums are the same ones: where the buffer is little
    wider than the rows the gradient lies alike, where it is twice as wide it is compact, and the bits are the same."""
    x = randn(m, v, seed=1, dtype=dtype, std=3)
    t, i = entries(m, v, 9, seed=2)
    w = randn(m, seed=3) > -1
    narrow, wide = v + 7 & -8, 2 * v + 7 & -8
    got = []
    for stride in (narrow, wide + 16):
        z = laid_out(x, stride).requires_grad_()
        loss = sft.distill_loss(z, t, i, row_weight=w)
        g, = torch.autograd.grad(loss, z, torch.ones_like(loss))
        got.append((loss.detach(), g))
    assert got[1][1].is_contiguous() and torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    check(laid_out(x, wide + 16), t, i, w=w)
