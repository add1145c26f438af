"""AdamW.load_state_dict keeps the buffers that a captured step names, without a GPU."""
import copy

import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200 import _lib


def begun(params, **kw):
    """An optimizer whose state is as a first step leaves it, with values in it."""
    opt = sft.AdamW(params, **kw)
    for group in opt.param_groups:
        for i, p in enumerate(group["params"]):
            st = opt._begin(p, group)
            for t in st.values():
                if isinstance(t, torch.Tensor):
                    t.copy_(torch.arange(t.numel()).view(t.shape) % 100 + i)
            st["step"] = 3
        if group["capturable"]:
            group["_counter"] = (torch.tensor([3]), torch.zeros(_lib.ADAMW_CONSTANTS, dtype=torch.uint8))
    return opt


def params(seed=0):
    return [torch.nn.Parameter(torch.full(s, float(seed))) for s in ((5000,), (40,), (8, 6))]


def places(opt):
    out = {}
    for g in opt.param_groups:
        for i, p in enumerate(g["params"]):
            out.update({(i, k): t.data_ptr() for k, t in opt.state[p].items() if isinstance(t, torch.Tensor)})
        if g.get("_counter") is not None:
            out["counter"], out["constants"] = (t.data_ptr() for t in g["_counter"])
    return out


@pytest.mark.parametrize("state", ["float32", "sf8"])
@pytest.mark.parametrize("capturable", [False, True])
def test_values_go_into_the_buffers_at_hand(state, capturable):
    opt = begun(params(), state=state, capturable=capturable)
    saved = copy.deepcopy(opt.state_dict())
    before = places(opt)
    for g in opt.param_groups:
        for p in g["params"]:
            for t in opt.state[p].values():
                if isinstance(t, torch.Tensor):
                    t.zero_()
            opt.state[p]["step"] = 9
        if capturable:
            g["_counter"][0].fill_(9)
    opt.load_state_dict(saved)
    assert places(opt) == before
    for p, st in zip(opt.param_groups[0]["params"], saved["state"].values()):
        assert opt.steps_done(p) == 3
        for k, t in st.items():
            assert torch.equal(opt.state[p][k], t) if isinstance(t, torch.Tensor) else opt.state[p][k] == t
    for st in saved["state"].values():                 # the values are copies: the saved ones are not written
        assert all(t.data_ptr() not in before.values() for t in st.values() if isinstance(t, torch.Tensor))


def test_a_new_optimizer_and_another_kind():
    opt = begun(params(), state="sf8", capturable=True)
    saved = opt.state_dict()
    new = sft.AdamW(params(), state="sf8", capturable=True)
    new.load_state_dict(saved)
    assert new.param_groups[0].get("_counter") is None and not set(places(new).values()) & set(places(opt).values())
    p = new.param_groups[0]["params"][0]
    assert new.state[p]["exp_avg"].dtype == torch.int8 and new.steps_done(p) == 3
    other = begun(params(), state="float32")
    other.load_state_dict(saved)                       # the saved kind of moments is what counts
    p = other.param_groups[0]["params"][0]
    assert other.state[p]["exp_avg"].dtype == torch.int8 and other.param_groups[0]["state"] == "sf8"


def test_float32_moments_take_the_parameters_layout():
    a, b = torch.nn.Parameter(torch.zeros(6, 8)), torch.nn.Parameter(torch.zeros(8, 6).t())
    saved = begun([a]).state_dict()
    opt = sft.AdamW([b])
    opt.load_state_dict(saved)
    for k in ("exp_avg", "exp_avg_sq"):
        assert opt.state[b][k].stride() == b.stride() and torch.equal(opt.state[b][k], saved["state"][0][k])


def test_a_state_of_before_the_first_step():
    """Saved before any step and loaded into an optimizer that may have been captured: zeros, in place."""
    fresh = sft.AdamW(params(), capturable=True).state_dict()
    opt = begun(params(), capturable=True)
    before = places(opt)
    opt.load_state_dict(fresh)
    assert places(opt) == before
    for p in opt.param_groups[0]["params"]:
        assert opt.steps_done(p) == 0 and all(not t.any() for t in opt.state[p].values() if isinstance(t, torch.Tensor))
    plain = begun(params())
    plain.load_state_dict(fresh)
    assert all(not plain.state.get(p) for p in plain.param_groups[0]["params"])


def test_a_state_of_another_setting():
    """Saved without capturable: the steps are counted on the host from there on."""
    saved = begun(params()).state_dict()
    opt = begun(params(), capturable=True)
    opt.param_groups[0]["_counter"][0].fill_(9)
    opt.load_state_dict(saved)
    assert not opt.param_groups[0]["capturable"] and all(opt.steps_done(p) == 3 for p in opt.param_groups[0]["params"])
    opt.state[opt.param_groups[0]["params"][0]]["step"] = 4
    assert opt.state_dict()["state"][0]["step"] == 4
