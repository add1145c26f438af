"""A convolution converted with accumulate="tensor": unfold, the tensor-core linear, and
its gradients, against the formula in 64 bits with the linear's own bounds."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import superfloat.python_b200.torch as sft
from test_gpu_tensor_linear import backward64, close, close_grad, codes64, forward64, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,conv", [
    ((2, 3, 17, 20), dict(out_channels=8, kernel_size=3, padding=1)),
    ((3, 8, 15, 9), dict(out_channels=21, kernel_size=(2, 3), stride=2, dilation=(1, 2), padding=(0, 2), bias=False)),
    ((1, 5, 6, 6), dict(out_channels=1, kernel_size=6)), ((4, 16, 8, 8), dict(out_channels=40, kernel_size=1))])
@pytest.mark.parametrize("scale", ["per_tensor", "per_channel"])
def test_a_convolution(gpu, shape, conv, dtype, scale):
    torch.manual_seed(0)
    plain = nn.Conv2d(shape[1], **conv).cuda().to(dtype)
    net = sft.convert(nn.Sequential(plain), dtype="sf8", accumulate="tensor", scale=scale)
    assert type(net[0]).__name__ == "SFConv2d"
    x = randn(*shape, seed=1, dtype=dtype).requires_grad_()
    y = net(x)
    assert y.shape == plain(x).shape and y.dtype == dtype
    dy = randn(*y.shape, seed=2, dtype=dtype)
    weight, bias = net[0].weight, net[0].bias
    wanted = [t for t in (x, weight, bias) if t is not None]
    gx, gw, *gb = torch.autograd.grad(y, wanted, dy)

    kw = dict(kernel_size=plain.kernel_size, dilation=plain.dilation, padding=plain.padding, stride=plain.stride)
    n = plain.out_channels
    rows = F.unfold(x.detach().double(), **kw).transpose(1, 2).flatten(0, 1)
    w = weight.detach().reshape(n, -1)
    codes, s = codes64(w, 8, scale)
    want, tol, _, _ = forward64(rows, codes, s, 8, bias, None, None)
    flat = lambda t: t.flatten(2).transpose(1, 2).flatten(0, 1)  # noqa: E731
    close(flat(y.detach()), want, tol, dtype)
    (dx, ex), dw, db = backward64(rows, codes, s, 8, bias, None, flat(dy), dtype, None, None)
    close_grad(gw.reshape(n, -1), dw, dtype)
    if bias is not None:
        close_grad(gb[0], db, dtype)
    # a pixel's gradient: the sum of its places in the rows, each rounded to the type, summed in float32, rounded
    half, taps = torch.finfo(dtype).eps / 2, rows.shape[1] // shape[1]
    fold = lambda t: F.fold(t.unflatten(0, (shape[0], -1)).transpose(1, 2), shape[2:], **kw)  # noqa: E731
    each = ex * (1 + half) + half * dx.abs() + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    close(gx, fold(dx), fold(each + taps * 2.0 ** -24 * dx.abs()), dtype)
