"""The distillation loss of rows whose largest logit, over the temperature, is far from 0: masks of a large finite value,
tiny temperatures, and rows of which some parts are far and some not.  The formula and its tolerances are those of
test_gpu_distill: an exponential's argument is off by 3 u |z| here too (a difference, the factor and their product)."""
import pytest
import torch

from test_gpu_distill import TYPES, check, entries, randn

pytestmark = pytest.mark.gpu
WIDTHS = [300, 9001, 50257]                        # one CTA and clusters


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", WIDTHS)
def test_rows_around_a_large_value(gpu, v, dtype):
    """Rows of one value (a share of 1 / V each), a few steps of the type around it, and one element above all others."""
    for at in (-1e30, -1e12, -1e10, -3e9, -1e9, 5e9, 1e12, 1e30, 1e36):
        x = torch.full((4, v), at, dtype=dtype, device="cuda")
        step = abs(at) * torch.finfo(dtype).eps
        x[1] += (randn(v, seed=1) * step).to(dtype)
        x[2, 7] = 0
        x[3, 3::5] = randn(len(range(3, v, 5)), seed=2, dtype=dtype)
        t, i = entries(4, v, 6, seed=3, absent=False)
        i[0, 0] = i[2, 3] = 7
        check(x, t, i, reduction="none", g=torch.ones(4, device="cuda"))
        check(x, t, i, T=2.5)


@pytest.mark.parametrize("v", WIDTHS)
def test_rows_at_the_border(gpu, v):
    """Values on both sides of 2^24 ln 2, a step of 1 apart, so that threads and CTAs of one row lie on either side."""
    border = 11629080.0
    for sign in (1.0, -1.0):
        x = sign * border + torch.randint(-9, 10, (5, v), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).float()
        x[1, : v // 2] = x[1, : v // 2].clamp(max=sign * border - 4)
        x[2, v // 2:] = x[2, v // 2:].clamp(max=sign * border - 4)
        x[3, 1:] -= 3e7
        x[4, 1:] -= 40
        t, i = entries(5, v, 9, seed=3, absent=False)
        check(x, t, i, reduction="none", g=torch.ones(5, device="cuda"))
        check(x, t, i, g=torch.tensor(2.0, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1e-6, 1e-5, 1e-3])
def test_small_temperatures(gpu, dtype, temperature):
    x = randn(6, 5003, dtype=dtype, std=20)
    x[3:] *= 50
    t, i = entries(6, 5003, 8, seed=2, absent=False)
    i[:, 0] = x.argmax(1)
    check(x, t, i, T=temperature, reduction="none", g=torch.ones(6, device="cuda"))
    check(x, t, i, T=temperature)
