"""The x's gradient in fp16 where the channels' scales are far apart: dz s is brought
within fp16's range by the largest scale of a channel that has a code other than 0."""
import pytest
import torch

import superfloat.python_b200.torch as sft
from test_gpu_tensor_linear import close_grad, backward64, randn

pytestmark = pytest.mark.gpu


def check(x, p, dy):
    """dx against the formula, the tolerance's step of the subnormals that of the largest scale with a code."""
    y = sft.tensor_linear(x, p)
    got, = torch.autograd.grad(y, x, dy)
    codes, s = p.codes.double(), p.scale.double()
    live = torch.where(codes.abs().amax(1) > 0, s, torch.zeros_like(s))
    pair = backward64(x, codes, live, 8, None, None, dy, torch.float16, None, None)[0]
    assert bool(got.isfinite().all())
    close_grad(got, pair, torch.float16)
    return got


@pytest.mark.parametrize("std", [2.0 ** -6, 2.0 ** -9])
@pytest.mark.parametrize("n,k", [(300, 40), (1500, 257), (130, 2000)])
def test_a_row_of_zeros_does_not_set_the_range(gpu, n, k, std):
    """A row of zeros (a pruned channel, a padded vocabulary) has the scale 1: dz s / 1 would be below fp16's normal range."""
    x = randn(20, k, dtype=torch.float16).requires_grad_()
    w = randn(n, k, seed=1, std=std)
    dy = randn(20, n, seed=2, std=2.0 ** -10, dtype=torch.float16)
    alive = check(x, sft.pack_weight(w), dy)
    w[n // 2], w[3], w[n - 1] = 0, 0, 0
    p = sft.pack_weight(w)
    assert float(p.scale[3]) == 1.0 and p.scale.sort().values[-4] < 0.1
    check(x, p, dy)
    check(x, p, (dy.float() * 2.0 ** 20).half())          # and large ones stay finite beside it
    w[n - 1, k - 1] = 127 / 128                           # the scale 1 with one code, the row's last
    p = sft.pack_weight(w)
    assert float(p.scale[n - 1]) == 1.0 and int(p.codes[n - 1].abs().max()) == 127
    check(x, p, dy)
    assert alive.shape == x.shape


@pytest.mark.parametrize("scale", [0.0, 2.0 ** -140, 2.0 ** -127])
def test_scales_at_the_end_of_the_range(gpu, scale):
    """Every scale 0 or below float32's normal range: dx is 0 in fp16, as the formula's."""
    x, dy = randn(20, 64, dtype=torch.float16).requires_grad_(), randn(20, 48, seed=2, dtype=torch.float16)
    p = sft.SFPackedWeight(sft.pack_weight(randn(48, 64, seed=1)).codes, torch.full((48,), scale, device="cuda"))
    assert float(check(x, p, dy).abs().max()) == 0


@pytest.mark.parametrize("w", [0.0, 1.0])
def test_all_rows_alike(gpu, w):
    x, dy = randn(20, 64, dtype=torch.float16).requires_grad_(), randn(20, 48, seed=2, dtype=torch.float16)
    check(x, sft.pack_weight(torch.full((48, 64), w, device="cuda")), dy)


def test_a_negative_scale(gpu):
    x, dy = randn(20, 64, dtype=torch.float16).requires_grad_(), randn(20, 48, seed=2, dtype=torch.float16)
    p = sft.pack_weight(randn(48, 64, seed=1, std=0.01))
    p.scale[::3] *= -1
    p.scale[5] = -1.0
    y = sft.tensor_linear(x, p)
    got, = torch.autograd.grad(y, x, dy)
    gx = backward64(x, p.codes.double(), p.scale.double(), 8, None, None, dy, torch.float16, None, None)[0]
    close_grad(got, gx, torch.float16)
