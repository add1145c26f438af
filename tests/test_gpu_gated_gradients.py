"""The gradients of a gated product's two weights are tensors of their own, although one product makes both."""
import pytest
import torch

import superfloat.python_b200.torch as sft
from test_gpu_tensor_linear import randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [64, 40])
@pytest.mark.parametrize("create_graph", [False, True])
def test_a_change_to_one_is_none_to_the_other(gpu, n, create_graph):
    x = randn(33, 48, dtype=torch.bfloat16)
    gate, up = (randn(n, 48, seed=s, dtype=torch.bfloat16).requires_grad_() for s in (1, 2))
    h = sft.tensor_gated(x, gate, up)
    dg, du = (t.detach() for t in torch.autograd.grad(h, (gate, up), torch.ones_like(h), create_graph=create_graph))
    want = du.clone()
    p = torch.ones_like(du, requires_grad=True)
    penalty = (p * du).sum()                           # (saves du)
    dg.mul_(2)
    dg.clamp_(-1, 1)
    assert torch.equal(torch.autograd.grad(penalty, p)[0], want) and torch.equal(du, want)
    assert dg.is_contiguous() and du.is_contiguous()
    h = sft.tensor_gated(x, gate, up)
    h.backward(torch.ones_like(h))
    kept = up.grad.clone()
    gate.grad.zero_()
    assert torch.equal(up.grad, kept) and torch.equal(kept, want)
