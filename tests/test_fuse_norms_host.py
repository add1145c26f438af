"""convert(fuse=True) on the host: a layer norm that the operator does not take, or that does more than its class, stays."""
import pytest
import torch
import torch.nn as nn

import superfloat.python_b200.torch as sft
from superfloat.python_b200 import _lib
from test_fuse_host import convert


def kept(norm):
    m = convert(nn.Sequential(norm))
    assert isinstance(m[0], nn.LayerNorm)
    return [why for path, _, why in sft.conversion_report(m).skipped if path == "0"][0]


def test_lengths():
    assert isinstance(convert(nn.Sequential(nn.LayerNorm(_lib.NORM_MOST)))[0], sft.SFLayerNorm)
    assert "65536 features" in kept(nn.LayerNorm(_lib.NORM_MOST + 1))
    with pytest.raises(ValueError, match="65536 features"):
        sft.SFLayerNorm(nn.LayerNorm(_lib.NORM_MOST + 1))
    assert "last dimension" in kept(nn.LayerNorm((3, 8)))


@pytest.mark.parametrize("kw", [dict(), dict(bias=False), dict(elementwise_affine=False)])
def test_parameters(kw):
    assert isinstance(convert(nn.Sequential(nn.LayerNorm(8, **kw)))[0], sft.SFLayerNorm)
    if "elementwise_affine" not in kw:
        assert "float64" in kept(nn.LayerNorm(8, **kw).double())


def test_what_does_more_than_its_class():
    class Doubled(nn.Module):
        def forward(self, w):
            return 2 * w

    norm = nn.LayerNorm(8)
    torch.nn.utils.parametrize.register_parametrization(norm, "weight", Doubled())
    assert "computed" in kept(norm)
    for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook"):
        norm = nn.LayerNorm(8)
        getattr(norm, register)(lambda *a: None)
        assert "hooks" in kept(norm)
    norm = nn.LayerNorm(8)
    norm.forward = lambda x: x
    assert "its own forward" in kept(norm)
