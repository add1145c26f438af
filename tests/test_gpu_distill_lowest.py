"""A teacher's entry where the student's logit is the type's lowest value, as masks leave it: the loss is T p times the
distance, finite wherever float32 holds that.  The formula and its tolerances are test_gpu_distill's."""
import pytest
import torch

import superfloat.python_b200.torch as sft
from test_gpu_distill import TYPES, check, entries, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1e-3, 0.5, 1.0, 2.5])
@pytest.mark.parametrize("v", [40, 9001, 50257])
def test_an_entry_at_the_lowest_value(gpu, v, temperature, dtype):
    x = randn(6, v, dtype=dtype, std=3)
    t, i = entries(6, v, 5, seed=2, absent=False)
    i[:] = torch.tensor([3, 5, 7, 11, 13], device="cuda")
    t[:, 4] = t[:, :4].amax(1) - 3 * temperature      # (a share of 5 % at most)
    low = torch.finfo(dtype).min
    x[1:, 13] = low
    x[2, 20:] = low
    x[3] -= 300
    x[3, 13] = low
    x[4, 12:] = low / 2
    for reduction in ("none", "mean"):
        loss, g = check(x, t, i, T=temperature, reduction=reduction, g=torch.ones(6 if reduction == "none" else (), device="cuda"))
        assert bool(loss.isfinite().all()) and bool(g.isfinite().all())
    assert dtype == torch.float16 or float(loss.detach()) > 1e30


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [40, 9001])
def test_a_row_with_an_infinity_is_not_a_number(gpu, v, dtype):
    x = randn(5, v, dtype=dtype, std=3)
    t, i = entries(5, v, 3, seed=2, absent=False)
    i[:] = torch.tensor([3, 5, 7], device="cuda")
    x[1, 2] = x[2, 3] = x[3, 5] = x[3, 6] = float("inf")
    x[3, 7] = torch.finfo(dtype).min
    x[4, 2], x[4, 3] = float("inf"), -float("inf")
    z = x.requires_grad_()
    loss = sft.distill_loss(z, t, i, reduction="none")
    g, = torch.autograd.grad(loss, z, torch.ones_like(loss))
    assert loss.isnan().tolist() == [False, True, True, True, True]
    assert bool(g[1:].isnan().all()) and not bool(g[0].isnan().any())
