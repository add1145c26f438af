"""A captured AdamW step goes on from a state that was loaded after the capture."""
import copy

import pytest
import torch

import superfloat.python_b200.torch as sft
from test_gpu_adamw import HYPER, backward, model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("state", ["float32", "sf8"])
def test_replays_after_a_load(gpu, state):
    net = model()
    params = list(net.parameters())
    opt = sft.AdamW(params, state=state, capturable=True, **HYPER)
    backward(net, 0)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()

    def run(n):
        for _ in range(n):
            graph.replay()
        torch.cuda.synchronize()
        return [p.detach().clone() for p in params] + [t.clone() for p in params for t in opt.moments(p)]

    start = run(2)
    saved = copy.deepcopy(opt.state_dict())
    want = run(3)
    assert all(opt.steps_done(p) == 6 for p in params)
    with torch.no_grad():
        for p, t in zip(params, start):
            p.copy_(t)
    opt.load_state_dict(saved)
    assert all(opt.steps_done(p) == 3 for p in params)
    noise = [torch.full_like(p, 7.0) for p in params * 4]     # what a freed buffer would have been given to
    got = run(3)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(bool((t == 7).all()) for t in noise)
    assert all(opt.steps_done(p) == 6 for p in params)


def test_capturable_turned_off_and_on(gpu):
    """The step count goes along: five steps in turns give what five of one kind give."""
    nets = [model() for _ in range(2)]
    opts = [sft.AdamW(n.parameters(), state="sf8", capturable=True, **HYPER) for n in nets]
    for i, on in enumerate([True, True, False, False, True]):
        opts[0].param_groups[0]["capturable"] = on
        for net, opt in zip(nets, opts):
            if i == 0:
                backward(net, 0)
            opt.step()
        for p, q in zip(*(n.parameters() for n in nets)):
            assert opts[0].steps_done(p) == opts[1].steps_done(q) == i + 1
    for p, q in zip(*(n.parameters() for n in nets)):
        # the moments have no constant that depends on the step; the update's two are a unit of float32 apart at most
        assert all(torch.equal(a, b) for a, b in zip(opts[0].moments(p), opts[1].moments(q)))
        off = float((p - q).detach().abs().max())
        assert off <= 5 * (2.0 ** -22 * HYPER["lr"] * 10 + 2.0 ** -23 * float(q.detach().abs().max()))
