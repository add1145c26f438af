"""pack() of gated blocks on the host: what is laid out, and a last projection of another arithmetic that stays as it is."""
import torch
import torch.nn as nn

import superfloat.python_b200.torch as sft
from superfloat.python_b200.torch import _tensor
from test_fuse_host import Gated, convert


def fake(w, dtype="sf8", scale="per_channel"):
    return sft.SFPackedWeight(torch.zeros(w.shape, dtype=torch.int8), torch.ones(w.shape[0]), dtype)


def test_a_last_projection_of_another_arithmetic_stays(monkeypatch):
    monkeypatch.setattr(_tensor, "pack_weight", fake)
    cfg = sft.SFConfig(8, "per_channel", accumulate="tensor")
    for down in (sft.SFConfig(16), sft.SFConfig(8, accumulate="chain"), sft.SFConfig(8, accumulate="wide")):
        block = sft.SFGatedFeedForward(Gated(), "b", cfg, down)
        for m in (sft.pack(block), sft.pack(nn.Sequential(block))[0]):
            assert isinstance(m, sft.SFPackedGatedFeedForward) and isinstance(m.gate_proj, sft.SFPackedLinear)
            assert isinstance(m.down_proj, sft.SFLinear) and m.down_proj.sf == down
    m = sft.pack(convert(nn.Sequential(Gated())))[0]
    assert isinstance(m.down_proj, sft.SFPackedLinear)
