"""sf::linear_tensor in traced training graphs, without a GPU: forward and backward
on tensors without memory, as torch.compile's training backends trace them."""
import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import superfloat.python_b200.torch as sft


@pytest.mark.parametrize("bias", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("want", ["xwb", "x", "w", "b"])
def test_gradients_of_tensors_without_memory(bias, want):
    with FakeTensorMode():
        x = torch.empty(5, 7, 64, dtype=torch.bfloat16, requires_grad="x" in want)
        w = torch.empty(24, 64, requires_grad="w" in want)
        b = None if bias is None else torch.empty(24, dtype=bias, requires_grad="b" in want)
        leaves = [t for t in (x, w, b) if t is not None and t.requires_grad]
        if not leaves:
            return
        y = torch.ops.sf.linear_tensor(x, w, b, 8, "per_tensor", "layer")
        assert y.shape == (5, 7, 24) and y.dtype == torch.bfloat16
        for g, t in zip(torch.autograd.grad(y, leaves, torch.empty_like(y)), leaves):
            assert g.shape == t.shape and g.dtype == t.dtype and g.device == t.device and g.is_contiguous()


def test_a_layer_traces_with_its_gradient():
    """A converted model's forward and backward pass as one graph: one node each way for a layer."""
    net = sft.convert(nn.Sequential(nn.Linear(64, 40), nn.GELU(), nn.Linear(40, 16, bias=False)).bfloat16(), dtype="sf6",
                      accumulate="tensor")
    params = dict(net.named_parameters())
    op = torch.ops.sf.linear_tensor

    def step(x, *values):
        ps = dict(zip(params, values))
        h = op(x, ps["0.weight"], ps["0.bias"], 6, "per_tensor", "0")
        y = op(nn.functional.gelu(h), ps["2.weight"], None, 6, "per_tensor", "2")
        return torch.autograd.grad(y.float().square().mean(), values)

    graph = make_fx(step, tracing_mode="fake")(torch.zeros(9, 64, dtype=torch.bfloat16), *params.values())
    names = [str(n.target) for n in graph.graph.nodes if "linear_tensor" in str(n.target)]
    assert sorted(names) == ["sf.linear_tensor.default"] * 2 + ["sf.linear_tensor_backward.default"] * 2
