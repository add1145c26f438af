"""Forward-mode derivatives of the tensor-core linear are refused, not dropped."""
import pytest
import torch
from torch.autograd import forward_ad

import superfloat.python_b200.torch as sft
from superfloat.python_b200 import _lib
from superfloat.python_b200._errors import SFShapeError, SFUnsupportedError
from superfloat.python_b200.torch import _tensor


def operands():
    return dict(x=torch.randn(200, 64).bfloat16(), weight=torch.randn(24, 64), bias=torch.randn(24),
                residual=torch.randn(200, 24).bfloat16())


@pytest.mark.parametrize("name", ["x", "weight", "bias", "residual"])
@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_of_each_operand(name, grad):
    args = operands()
    args["bias"].requires_grad_(grad and name != "bias")
    with forward_ad.dual_level():
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(SFUnsupportedError, match="forward-mode"):
            sft.tensor_linear(**args, activation="gelu")


def test_a_packed_weight_and_the_layers():
    args = operands()
    with forward_ad.dual_level():
        x = forward_ad.make_dual(args["x"], torch.ones_like(args["x"]))
        scale = forward_ad.make_dual(torch.ones(24), torch.ones(24))
        codes = torch.zeros(24, 64, dtype=torch.int8)
        for packed, inp in ((sft.SFPackedWeight(codes, scale), args["x"]), (sft.SFPackedWeight(codes, torch.ones(24)), x)):
            with pytest.raises(SFUnsupportedError, match="forward-mode"):
                sft.tensor_linear(inp, packed)
        layer = sft.convert(torch.nn.Linear(64, 24).bfloat16(), dtype="sf8", accumulate="tensor")
        for call in (lambda: layer(x), lambda: torch.ops.sf.linear_tensor(x, args["weight"], None, 8, "per_tensor", "layer")):
            with torch.no_grad(), pytest.raises(SFUnsupportedError, match="forward-mode"):
                call()


def test_operands_without_a_tangent_pass(monkeypatch):
    """Within a dual level, and outside of one, plain operands reach the other checks."""
    args = operands()
    with forward_ad.dual_level(), pytest.raises(SFShapeError, match="CUDA"):
        sft.tensor_linear(**args)
    with pytest.raises(SFShapeError, match="CUDA"):
        sft.tensor_linear(**args)
    monkeypatch.setattr(_lib, "tensor_forward", lambda index, call: None)
    monkeypatch.setattr(_tensor, "_check_weight", lambda w: None)
    monkeypatch.setattr(_tensor, "_check_operands", lambda *a: None)
    with pytest.raises(Exception):                     # functorch's tensors have no memory of their own
        torch.func.jvp(lambda x: sft.tensor_linear(x, args["weight"]), (args["x"],), (args["x"],))
