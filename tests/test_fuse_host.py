"""convert(fuse=True) and pack() on the host: which blocks become one operator, which do not and why."""
import copy

import pytest
import torch
import torch.nn as nn

import superfloat.python_b200.torch as sft


class Gated(nn.Module):
    def __init__(self, d=16, h=24, act=None, bias=False):
        super().__init__()
        self.gate_proj, self.up_proj = nn.Linear(d, h, bias=bias), nn.Linear(d, h, bias=bias)
        self.down_proj, self.act_fn = nn.Linear(h, d, bias=bias), act or nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Swapped(Gated):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.up_proj(x)) * self.gate_proj(x))


class Block(nn.Module):
    def __init__(self, **kw):
        super().__init__()
        self.norm, self.mlp, self.head = nn.LayerNorm(16), Gated(**kw), nn.Linear(16, 32)

    def forward(self, x):
        return self.head(x + self.mlp(self.norm(x)))


def convert(net, **kw):
    return sft.convert(net, dtype="sf8", accumulate="tensor", scale="per_channel", fuse=True, **kw)


@pytest.mark.parametrize("act,name", [(nn.SiLU(), "silu"), (nn.GELU(), "gelu"), (nn.GELU(approximate="tanh"), "gelu_tanh"), (nn.ReLU(), "relu")])
def test_blocks_become_one_operator(act, name):
    net = Block(act=act, bias=True)
    m = convert(net)
    assert isinstance(m.norm, sft.SFLayerNorm) and isinstance(m.mlp, sft.SFGatedFeedForward) and m.mlp.activation == name
    assert isinstance(m.mlp.down_proj, sft.SFLinear) and isinstance(m.head, sft.SFLinear)
    assert set(m.state_dict()) == set(net.state_dict()) and type(net.mlp) is Gated
    kinds = dict(sft.conversion_report(m).converted)
    assert kinds["mlp"] == "gated feed-forward" and kinds["norm"] == "LayerNorm"
    assert set(sft.conversion_report(m).widths) == {"mlp.gate_proj", "mlp.up_proj", "mlp.down_proj", "head"}
    # the parameters are the source's own
    own = convert(net, inplace=True)
    assert own.mlp.gate_proj.weight is net.mlp.gate_proj.weight and own.norm.eps == 1e-5
    again = convert(own)
    assert isinstance(again.mlp, sft.SFGatedFeedForward) and type(again.mlp.gate_proj) is nn.Linear


def test_widths_and_what_is_not_one_operator():
    m = convert(Block(), widths={"mlp.gate_proj": "sf6", "mlp.up_proj": "sf6"})
    assert m.mlp.sf.bits == 6 and m.mlp.down_proj.sf.bits == 8
    m = convert(Block(), widths={"mlp.gate_proj": "sf6"})
    assert type(m.mlp) is Gated and m.mlp.gate_proj.sf.bits == 6 and m.mlp.up_proj.sf.bits == 8
    for block, why in ((Swapped(), "something else"), (Gated(act=nn.Tanh()), "activation Tanh")):
        net = nn.Sequential(block, nn.LayerNorm((4, 16)))
        m = convert(net)
        report = sft.conversion_report(m)
        assert type(m[0]) is type(block) and isinstance(m[0].gate_proj, sft.SFLinear) and type(m[1]) is nn.LayerNorm
        assert any(why in reason for _, _, reason in report.skipped), report
    odd = Gated()
    odd.up_proj = nn.Linear(16, 24).double()
    odd.extra = nn.Dropout()
    assert type(convert(nn.Sequential(odd))[0]) is Gated
    plain = sft.convert(Block(), dtype="sf8", accumulate="tensor")
    assert type(plain.mlp) is Gated and type(plain.norm) is nn.LayerNorm
    with pytest.raises(ValueError, match="fuse"):
        sft.convert(Block(), dtype="sf8", fuse=True)


def test_shared_blocks_and_copies():
    mlp = Gated()
    net = nn.Sequential(mlp, mlp)
    m = convert(net)
    assert m[0] is m[1] and sft.conversion_report(m).shared == [("1", "0")]
    c = copy.deepcopy(m)
    assert c[0] is c[1] and c[0] is not m[0]
    assert convert(Gated()).activation == "silu"              # the model is the block


def test_a_norm_refuses_other_rows():
    m = convert(Block())
    from superfloat.python_b200._errors import SFShapeError
    with pytest.raises(SFShapeError, match="16 features"):
        m.norm(torch.zeros(3, 8))
    with pytest.raises(ValueError, match="last dimension"):
        sft.SFLayerNorm(nn.LayerNorm((3, 4)))
