"""An AdamW step happens as a whole or not at all: what is refused in one of a call's
launches leaves the tensors of the others as they were."""
import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200._errors import SFError, SFShapeError
from test_gpu_adamw import HYPER, make

pytestmark = pytest.mark.gpu


def views(dtype):
    """Two parameters that overlap by 100 elements, their gradients and moments."""
    wide = torch.ones(900, dtype=dtype, device="cuda")
    return [wide[:500], wide[400:]]


def snapshot(tensors):
    return [(t.detach().clone(), t._version) for t in tensors]


def check_unchanged(tensors, before):
    same = [torch.equal(t, old) and t._version == version for t, (old, version) in zip(tensors, before)]
    assert all(same), same


@pytest.mark.parametrize("kinds", [("f32", "f32"), ("f32", "sf8"), ("sf8", "f32")])
def test_a_refusal_in_the_second_launch(gpu, kinds):
    """A float32 tensor and two overlapping bf16 ones: two launches, of which the second cannot be."""
    p, g, m, v = make([5000], torch.float32)
    over = views(torch.bfloat16)
    p, g = p + over, g + [torch.ones_like(t) for t in over]
    moments = lambda kind, n: (sft.SF8Moment.zeros(n, "cuda") if kind == "sf8" else  # noqa: E731
                               torch.zeros(n, device="cuda"))
    m, v = ([moments(kinds[min(i, 1)], t.numel()) for i, t in enumerate(p)] for _ in range(2))
    flat = [u for t in m + v for u in ((t.codes, t.scale) if isinstance(t, sft.SF8Moment) else (t,))]
    before = snapshot(p + flat)
    for order in ([0, 1, 2], [1, 2, 0], [1, 0, 2]):
        args = [[x[i] for i in order] for x in (p, g, m, v)]
        with pytest.raises(SFError, match="overlaps"):
            sft.adamw_step(*args, step=1, **HYPER)
        check_unchanged(p + flat, before)


@pytest.mark.parametrize("capturable", [False, True])
def test_a_refusal_in_the_second_group(gpu, capturable):
    """AdamW's groups: the first one's parameters, moments and step count stay."""
    a = torch.nn.Parameter(torch.ones(5000, device="cuda"))
    b, c = (torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2))
    opt = sft.AdamW([{"params": [a]}, {"params": [b, c]}], state="sf8", capturable=capturable, **HYPER)
    for p in (a, b, c):
        p.grad = torch.ones_like(p)
    opt.step()
    b.data = c.data
    kept = [t for q in (a, b, c) for t in (q, *(s for s in opt.state[q].values() if isinstance(s, torch.Tensor)))]
    before, done = snapshot(kept), [opt.steps_done(q) for q in (a, b, c)]
    with pytest.raises(SFShapeError, match="given twice"):
        opt.step()
    check_unchanged(kept, before)
    assert [opt.steps_done(q) for q in (a, b, c)] == done == [1, 1, 1]
    whole = torch.ones(500, device="cuda")
    b.data, c.data = whole[:300], whole[200:]
    kept = [t for q in (a, b, c) for t in (q, *(s for s in opt.state[q].values() if isinstance(s, torch.Tensor)))]
    before = snapshot(kept)
    with pytest.raises(SFError, match="overlaps"):
        opt.step()
    check_unchanged(kept, before)
    assert [opt.steps_done(q) for q in (a, b, c)] == done
    c.data = torch.ones(300, device="cuda")
    opt.step()
    assert [opt.steps_done(q) for q in (a, b, c)] == [2, 2, 2]


def test_a_bad_setting_or_gradient_of_the_second_group(gpu):
    a, b = (torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2))
    opt = sft.AdamW([{"params": [a]}, {"params": [b]}], **HYPER)
    for p in (a, b):
        p.grad = torch.ones_like(p)
    before = snapshot([a, b])
    opt.param_groups[1]["lr"] = -1.0
    with pytest.raises(ValueError, match="lr"):
        opt.step()
    check_unchanged([a, b], before)
    opt.param_groups[1]["lr"] = 0.1
    b.data = b.data.double()
    b.grad = torch.ones_like(b)
    with pytest.raises(SFError, match="float64"):
        opt.step()
    assert torch.equal(a, before[0][0]) and a._version == before[0][1] and opt.steps_done(a) == 0
