"""The tensor-core products launched one straight after another (many short ones,
whose barriers' last arrivals come near the end of their CTAs), and over very many rows.
"""
import pytest
import torch

import superfloat.python_b200.torch as sft
from test_gpu_tensor_linear import backward64, close_grad, codes64, randn

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


@pytest.mark.parametrize("n,act,wscale", [(8, "gelu", "per_channel"), (5, None, "per_channel"), (8, "silu", "per_tensor")])
def test_gradients_of_very_many_rows(gpu, n, act, wscale):
    """More than 65535 x 64 rows, as a convolution of 64 images of 256 x 256 has them: the first gradient's blocks pass
    what a grid's second and third dimensions hold."""
    m, k, dtype = 65535 * 64 + 135, 8, torch.bfloat16
    x = randn(m, k, dtype=dtype).requires_grad_()
    w, b = randn(n, k, seed=1, std=0.3).requires_grad_(), randn(n, seed=2).requires_grad_()
    dy = randn(m, n, seed=3, dtype=dtype)
    y = sft.tensor_linear(x, w, b, activation=act, scale=wscale)
    grads = torch.autograd.grad(y, [x, w, b], dy)
    codes, s = codes64(w, 8, wscale)
    for got, pair in zip(grads, backward64(x, codes, s, 8, b, act, dy, dtype, w.dtype, None)):
        close_grad(got, pair, got.dtype)
    # the bias's gradient alone: a kernel adds its sums up
    alone = sft.tensor_linear(x.detach(), w.detach(), b, activation=act, scale=wscale)
    assert torch.equal(torch.autograd.grad(alone, b, dy)[0], grads[2])
