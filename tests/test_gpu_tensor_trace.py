"""Converted layers of accumulate="tensor" trained through torch.compile's tracing
backends: the eager layers' results and gradients, bit for bit."""
import pytest
import torch
import torch.nn as nn

import superfloat.python_b200.torch as sft
from superfloat.python_b200._errors import SFShapeError
from test_gpu_tensor_linear import randn
from test_gpu_tensor_training import batch, loss_of, model

pytestmark = pytest.mark.gpu


def test_a_compiled_training_step(gpu):
    """Three layers, an embedding and a residual: forward and backward as two traced graphs, without a break."""
    net, ids = model(scale="per_tensor"), batch()
    with torch.no_grad():
        net.up.weight[7] = 0
    loss_of(net, ids).backward()
    want = {n: p.grad.clone() for n, p in net.named_parameters()}
    net.zero_grad()
    logits = torch.compile(net, backend="aot_eager", fullgraph=True)(ids[:, :-1])
    nn.functional.cross_entropy(logits.flatten(0, 1).float(), ids[:, 1:].flatten()).backward()
    for n, p in net.named_parameters():
        assert torch.equal(p.grad, want[n]), n


@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (7, 40, 24), (90, 33, 41), (300, 130, 64)])
@pytest.mark.parametrize("wscale", ["per_channel", "per_tensor"])
def test_the_gradient_op(gpu, m, n, k, wscale):
    """Each set of gradients, rows with gaps and a transposed weight, beside tensor_linear's own."""
    x, w = randn(m, k + 8, dtype=torch.float16)[:, :k], randn(k, n, seed=1, std=k ** -0.5).t()
    b, dy = randn(n, seed=2), randn(m, n, seed=3, dtype=torch.float16)
    for wants in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        for bias in (b, None):
            if bias is None and wants[2]:
                continue
            leaves = [None if t is None else t.detach().requires_grad_(bool(want)) for t, want in zip((x, w, bias), wants)]
            wanted = [t for t in leaves if t is not None and t.requires_grad]
            got = torch.autograd.grad(torch.ops.sf.linear_tensor(*leaves, 8, wscale, "layer"), wanted, dy)
            want = torch.autograd.grad(sft.tensor_linear(*leaves, scale=wscale), wanted, dy)
            assert all(torch.equal(p, q) and p.dtype == q.dtype for p, q in zip(got, want))


def test_no_rows_and_a_second_derivative(gpu):
    x = torch.zeros(2, 0, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w, b = randn(20, 16).requires_grad_(), randn(20).requires_grad_()
    gx, gw, gb = torch.autograd.grad(torch.ops.sf.linear_tensor(x, w, b, 8, "per_tensor", "layer").sum(), [x, w, b])
    assert gx.shape == x.shape and float(gw.abs().sum()) == 0 and float(gb.abs().sum()) == 0
    x = randn(20, 16, dtype=torch.bfloat16).requires_grad_()
    y = torch.ops.sf.linear_tensor(x, w, b, 8, "per_tensor", "layer")
    g, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="autograd formula|differentiate"):
        g.float().sum().backward()


def test_the_gradient_op_refuses_what_does_not_fit(gpu):
    """Called by hand: a gradient of another size, type or device than the result's is refused before a launch."""
    x, w, g = randn(20, 16, dtype=torch.bfloat16), randn(24, 16), randn(20, 24, seed=1, dtype=torch.bfloat16)
    op = torch.ops.sf.linear_tensor_backward
    for bad in (g[:19], g[:, :23], g.float(), g.cpu(), g[None]):
        with pytest.raises(SFShapeError, match="gradient"):
            op(bad, x, w, None, 8, "per_tensor", True, True, False)
    with pytest.raises(SFShapeError, match="no bias"):
        op(g, x, w, None, 8, "per_tensor", True, True, True)
    with pytest.raises(SFShapeError, match="features"):
        op(g, x[:, :8], w, None, 8, "per_tensor", True, True, False)
    gx, gw, gb = op(g, x, w, None, 8, "per_tensor", True, False, False)
    assert gx.shape == x.shape and gw.numel() == 0 and gb.numel() == 0
