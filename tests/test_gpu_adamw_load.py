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
