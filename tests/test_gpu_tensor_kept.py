"""The tensor-core linear's gradients where x has gaps between its rows, and where
saved-tensor hooks (activation offloading) hand back what was kept in another
layout: the bits of the plain call."""
import pytest
import torch
import torch.utils.checkpoint

import superfloat.python_b200.torch as sft
from test_gpu_tensor_linear import backward64, close_grad, codes64, randn

pytestmark = pytest.mark.gpu


def compact(t):
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def odd(t):
    wide = torch.empty(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)[..., 1:1 + t.shape[-1]]
    return wide.copy_(t)


def gradients(x, w, b, r, dy, act, wscale):
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]     # x keeps its strides
    assert leaves[0].stride() == x.stride()
    y = sft.tensor_linear(*leaves, activation=act, residual=r, scale=wscale)
    return leaves, y, lambda: torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,wide,at", [(700, 256, 300, 768, 256), (130, 64, 96, 200, 8), (90, 40, 33, 41, 1),
                                           (65, 13, 40, 16, 0), (1, 24, 16, 96, 24), (300, 1, 8, 8, 0)])
def test_gradients_of_rows_with_gaps(gpu, dtype, m, k, n, wide, at):
    """A slice of a wider buffer, as a fused projection's result is sliced, against the formula and the dense call."""
    x = randn(m, wide, dtype=dtype)[:, at:at + k]
    w, b, dy = randn(n, k, seed=1, std=k ** -0.5), randn(n, seed=2), randn(m, n, seed=3, dtype=dtype)
    for wscale in ("per_channel", "per_tensor"):
        for act in (None, "gelu"):
            leaves, y, grads = gradients(x, w, b, None, dy, act, wscale)
            got = grads()
            want = gradients(x.contiguous(), w, b, None, dy, act, wscale)[2]()
            assert all(torch.equal(p, q) for p, q in zip(got, want))
            codes, s = codes64(w, 8, wscale)
            for p, pair in zip(got, backward64(x, codes, s, 8, b, act, dy, dtype, w.dtype, None)):
                close_grad(p, pair, p.dtype)


@pytest.mark.parametrize("m,k,n,wide", [(700, 256, 300, 768), (700, 256, 300, 256), (90, 40, 33, 41), (65, 13, 40, 13),
                                        (1, 24, 16, 96)])
def test_kept_tensors_in_another_layout(gpu, m, k, n, wide):
    x = randn(m, wide, dtype=torch.bfloat16)[:, :k]
    w, b, dy = randn(n, k, seed=1, std=k ** -0.5), randn(n, seed=2), randn(m, n, seed=3, dtype=torch.bfloat16)
    r = randn(m, n, seed=4, dtype=torch.bfloat16)
    hooks = [lambda: torch.autograd.graph.save_on_cpu(), lambda: torch.autograd.graph.save_on_cpu(pin_memory=True)]
    hooks += [lambda how=how: torch.autograd.graph.saved_tensors_hooks(how, lambda t: t) for how in (compact, odd, turned_here)]
    for wscale in ("per_channel", "per_tensor"):
        for act in (None, "silu"):
            want = gradients(x, w, b, r, dy, act, wscale)[2]()
            for hook in hooks:
                with hook():
                    grads = gradients(x, w, b, r, dy, act, wscale)[2]
                assert all(torch.equal(p, q) for p, q in zip(grads(), want))


def turned_here(t):
    return compact(t.t()).t() if t.dim() == 2 else compact(t)


def test_a_packed_weight_and_a_checkpointed_layer(gpu):
    x = randn(200, 96, dtype=torch.bfloat16)[:, :64]
    p, b = sft.pack_weight(randn(48, 64, seed=1, std=0.1)), randn(48, seed=2)
    dy = randn(200, 48, seed=3, dtype=torch.bfloat16)

    def run(wrap):
        leaves = [x.detach().requires_grad_(), b.detach().requires_grad_()]
        y = wrap(lambda x, b: sft.tensor_linear(x, p, b, activation="gelu_tanh"), *leaves)
        return y.detach(), *torch.autograd.grad(y, leaves, dy)

    want = run(lambda f, *a: f(*a))
    with torch.autograd.graph.save_on_cpu():
        again = run(lambda f, *a: f(*a))
    redone = run(lambda f, *a: torch.utils.checkpoint.checkpoint(f, *a, use_reentrant=False))
    for got in (again, redone):
        assert all(torch.equal(p, q) for p, q in zip(got, want))
