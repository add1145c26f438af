"""convert(fuse=True) on the host: a block becomes one operator only where its forward is down(act(gate(x)) * up(x)) and
nothing else, whatever its weights, its mode and the values on which it is tried."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import superfloat.python_b200.torch as sft
from test_fuse_host import Gated, Swapped, convert


class Clamped(Gated):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x).clamp(max=7e30)) * self.up_proj(x).clamp(min=-7e30, max=7e30))


class Dropped(Gated):
    def forward(self, x):
        return self.down_proj(F.dropout(self.act_fn(self.gate_proj(x)) * self.up_proj(x), 0.1, self.training))


class DroppedInTraining(Gated):
    def forward(self, x):
        h = self.act_fn(self.gate_proj(x)) * self.up_proj(x)
        return self.down_proj(F.dropout(h, 0.1) if self.training else h)


class OnlyWithGradients(Gated):
    def forward(self, x):
        h = self.act_fn(self.gate_proj(x)) * self.up_proj(x)
        return self.down_proj(h * 0.5 if torch.is_grad_enabled() else h)


class Held(Gated):
    def forward(self, x):
        with torch.no_grad():
            g = self.act_fn(self.gate_proj(x))
        return self.down_proj(g * self.up_proj(x))


class InAnotherType(Gated):
    def forward(self, x):
        with torch.autocast("cpu", torch.bfloat16):
            return super().forward(x)


class Halved(Gated):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x) * 0.5)


class ByValue(Gated):
    def forward(self, x):
        h = self.act_fn(self.gate_proj(x)) * self.up_proj(x)
        return self.down_proj(h.clamp(max=9) if bool(h.max() > 1e6) else h)


class ByLength(Gated):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * (self.up_proj(x) if len(x) < 100 else self.gate_proj(x)))


class Within(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x + 0

    @staticmethod
    def backward(ctx, g):
        return g


class OwnNode(Gated):
    def forward(self, x):
        return self.down_proj(Within.apply(self.act_fn(self.gate_proj(x)) * self.up_proj(x)))


class Residual(Gated):
    def forward(self, x):
        return x + self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Scaled(Gated):
    """(the factor is 1 when the block is converted)"""

    def __init__(self):
        super().__init__()
        self.factor = nn.Parameter(torch.ones(()))

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x)) * self.factor


class ByBuffer(Gated):
    def __init__(self):
        super().__init__()
        self.register_buffer("limit", torch.tensor(9.0))


class TwoArguments(Gated):
    def forward(self, x, residual=None):
        y = self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))
        return y if residual is None else y + residual


class ReLU(nn.Module):
    """(Another's name.)"""

    def forward(self, x):
        return F.relu(x) ** 2


class Sharper(nn.GELU):
    def forward(self, x):
        return F.gelu(2 * x)


class Plain(Gated):
    """Other ways to write the same."""

    def forward(self, hidden):
        h = self.up_proj(hidden)
        h *= self.act_fn(self.gate_proj(hidden))
        return self.down_proj(h)


def reason(block):
    m = convert(nn.Sequential(block))
    assert not isinstance(m[0], sft.SFGatedFeedForward) and isinstance(m[0].gate_proj, sft.SFLinear)
    return [why for path, _, why in sft.conversion_report(m).skipped if path == "0"][0]


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("kind", [Clamped, Dropped, DroppedInTraining, OnlyWithGradients, Held, InAnotherType, Halved, ByValue, ByLength, OwnNode,
                                  Residual])
def test_a_forward_that_does_something_else(kind, training):
    assert "something else" in reason(kind().train(training))


@pytest.mark.parametrize("act", [nn.SiLU(), nn.GELU(), nn.ReLU()])
@pytest.mark.parametrize("zero", ["down_proj", "up_proj", "gate_proj"])
def test_weights_of_zero_hide_nothing(zero, act):
    for kind in (Swapped, Halved, Clamped):
        block = kind(act=act, bias=True)
        nn.init.zeros_(getattr(block, zero).weight)
        nn.init.zeros_(getattr(block, zero).bias)
        assert "something else" in reason(block)
    plain = Gated(act=act)
    nn.init.zeros_(getattr(plain, zero).weight)
    assert isinstance(convert(nn.Sequential(plain))[0], sft.SFGatedFeedForward)


@pytest.mark.parametrize("act", [ReLU(), Sharper(), nn.Tanh(), nn.Sequential(nn.SiLU()), nn.SiLU(), nn.GELU(), torch.tanh, None])
def test_an_activation_is_what_it_computes(act):
    block = Gated()
    del block._modules["act_fn"]
    block.act_fn = act
    known = isinstance(act, (nn.SiLU, nn.Sequential)) or type(act) is nn.GELU
    if known:
        assert convert(nn.Sequential(block))[0].activation == ("gelu" if type(act) is nn.GELU else "silu")
    else:
        assert "activation" in reason(block)


def test_state_hooks_and_arguments():
    assert "parameters or buffers" in reason(Scaled()) and "parameters or buffers" in reason(ByBuffer())
    assert "one argument" in reason(TwoArguments())
    for where in ("gate_proj", "up_proj", "act_fn", None):
        for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook"):
            block = Gated()
            getattr(block if where is None else getattr(block, where), register)(lambda *a: None)
            assert "hooks" in reason(block)


@pytest.mark.parametrize("training", [True, False])
def test_the_same_written_otherwise(training):
    for act in (nn.SiLU(), nn.SiLU(inplace=True), nn.ReLU(inplace=True)):
        for kind in (Gated, Plain):
            block = kind(act=act).train(training)
            block.act_fn.eval()
            m = convert(nn.Sequential(block))[0]
            assert isinstance(m, sft.SFGatedFeedForward) and m.activation == ("relu" if type(act) is nn.ReLU else "silu")
            assert block.training is training and block.up_proj.training is training and not block.act_fn.training
    tied = Gated()
    tied.up_proj.weight = tied.gate_proj.weight
    assert isinstance(convert(nn.Sequential(tied))[0], sft.SFGatedFeedForward)
    same = Swapped()
    same.up_proj = same.gate_proj
    assert isinstance(convert(nn.Sequential(same))[0], sft.SFGatedFeedForward)


def test_a_block_runs_no_more_often_than_it_is_asked():
    """Once in each mode, not again by the module that stands for it; no random numbers are drawn."""
    class Counted(Gated):
        runs = 0

        def forward(self, x):
            Counted.runs += 1
            return super().forward(x)

    state = torch.get_rng_state()
    block = Counted()
    state = torch.get_rng_state()
    assert isinstance(convert(nn.Sequential(block), inplace=True)[0], sft.SFGatedFeedForward)
    assert Counted.runs == 4 and torch.equal(torch.get_rng_state(), state)


def test_inference_mode():
    with torch.inference_mode():
        block = Gated()
        assert isinstance(convert(nn.Sequential(block))[0], sft.SFGatedFeedForward)
        assert "something else" in reason(Clamped())
    assert isinstance(convert(nn.Sequential(block), inplace=True)[0], sft.SFGatedFeedForward)


@pytest.mark.parametrize("where", ["gate_proj", "up_proj", "act_fn", None])
def test_a_forward_set_on_the_module(where):
    block = Gated()
    m = block if where is None else getattr(block, where)
    own, seen = m.forward, []
    m.forward = lambda x: (seen.append(1), own(x))[1]
    assert "hooks" in reason(block)
