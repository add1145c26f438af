"""The tensor-core products launched one straight after another: many short ones,
whose barriers' last arrivals come near the end of their CTAs."""
import pytest
import torch

import superfloat.python_b200.torch as sft
from test_gpu_tensor_linear import randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(49, 8, 8), (49, 300, 64), (300, 40, 130), (129, 2100, 385), (700, 3000, 449)])
def test_short_products_back_to_back(gpu, m, n, k, dtype):
    """From one stage of the contraction to more than the ring of stages holds, on two streams: each call's bits are
    the first one's, and no wait runs out."""
    before = sft.tensor_failures()
    x = randn(m, k, dtype=dtype).requires_grad_()
    w = randn(n, k, seed=1, std=k ** -0.5).requires_grad_()
    dy = randn(m, n, seed=2, dtype=dtype)

    def step():
        y = sft.tensor_linear(x, w, activation="silu")
        return (y.detach(), *torch.autograd.grad(y, [x, w], dy))

    want, streams, got = step(), [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))
    assert sft.tensor_failures() == before
