"""The AdamW step on the B200 against its formula in 64 bits.

Tolerances, per element: the parameter is rounded once in its type (half a
step, eps / 2 of the value); the float32 arithmetic before that has the
roundings of p (1 - lr wd) and of the difference (2^-24 each of |p|) and the
quotient's: 6 roundings and two approximate operations within 2 units each,
under 2^-20 of the update as it would be without cancellation: where b1 m and
(1 - b1) g nearly cancel, their rounding errors, 3 x 2^-24 of T = b1 |m| +
(1 - b1) |g|, stay while m1 gets small, so the update's error is bounded by
2^-20 (lr / bc1) T / (sqrt(v / bc2) + eps) and not by 2^-20 of the update.
float32 moments: two products and a sum, under 4 x 2^-24 of the terms'
magnitudes.  sf8 codes equal the float32 restatement bit for bit.
"""
import numpy as np
import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200._errors import SFShapeError, SFTypeError, SFUnsupportedError
from test_adamw_host import BLOCK, dither, moment_codes, moment_values, step_f32

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [1, 3, 4, 255, 256, 257, 4095, 4096, 4097, 70001]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(sizes, dtype, seed=0):
    g = gen(seed)
    rnd = lambda n, s: torch.randn(n, generator=g, device="cuda") * s  # noqa: E731
    p = [rnd(n, 0.1).to(dtype) for n in sizes]
    gr = [rnd(n, 0.01).to(dtype) for n in sizes]
    m = [rnd(n, 0.003) for n in sizes]
    v = [rnd(n, 0.01).square() for n in sizes]
    return p, gr, m, v


def formula(p, g, m, v, step):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    b1, b2 = HYPER["betas"]
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    rate = HYPER["lr"] / (1 - b1 ** step) / (torch.sqrt(v1 / (1 - b2 ** step)) + HYPER["eps"])
    up = rate * (b1 * m.abs() + (1 - b1) * g.abs())              # without cancellation: the tolerance's measure
    return p * (1 - HYPER["lr"] * HYPER["weight_decay"]) - rate * m1, m1, v1, up


def check_p(got, want, update, before, dtype):
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tol = half * want.abs() + 2 * 2.0 ** -24 * (before.double().abs() + want.abs()) + 2.0 ** -20 * update.abs()
    tol = tol + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", TYPES)
def test_f32_states(gpu, dtype):
    p, g, m, v = make(SIZES, dtype)
    old = [[t.clone() for t in x] for x in (p, g, m, v)]
    assert sft.adamw_step(p, g, m, v, step=7, **HYPER) is None
    for i in range(len(SIZES)):
        want, m1, v1, up = formula(*(x[i] for x in old), 7)
        check_p(p[i], want, up, old[0][i], dtype)
        b1, b2 = HYPER["betas"]
        terms = b1 * old[2][i].double().abs() + (1 - b1) * g[i].double().abs()
        assert bool(((m[i].double() - m1).abs() <= 4 * 2.0 ** -24 * terms).all())
        assert bool(((v[i].double() - v1).abs() <= 4 * 2.0 ** -24 * v1).all())
        assert torch.equal(g[i], old[1][i])


def host(t):
    return t.detach().float().cpu().numpy()


@pytest.mark.parametrize("dtype", TYPES)
def test_sf8_states_bit_for_bit(gpu, dtype):
    """Three steps from zero states: codes and scales equal the restatement's, the parameter its formula."""
    p, g, _, _ = make(SIZES, dtype, 3)
    for t in g:
        t.mul_(torch.rand(t.shape, generator=gen(5), device="cuda") ** 4)     # a wide range within a block
    g[6][256:600] = 0
    mm = [sft.SF8Moment.zeros(n, "cuda") for n in SIZES]
    vv = [sft.SF8Moment.zeros(n, "cuda") for n in SIZES]
    ref = [(np.zeros(n, np.int8), np.zeros(-(-n // BLOCK), np.float32)) * 2 for n in SIZES]
    for step in (1, 2, 3):
        before = [t.clone() for t in p]
        sft.adamw_step(p, g, mm, vv, step=step, dither=11 * step, **HYPER)
        for i, n in enumerate(SIZES):
            mc, ms, vc, vs = ref[i]
            m0, v0 = moment_values(mc, ms, 2), moment_values(vc, vs, 4)
            want, m1, v1 = step_f32(host(before[i]), host(g[i]), m0, v0, step, HYPER["lr"], HYPER["betas"],
                                    HYPER["eps"], HYPER["weight_decay"])
            um, uv = dither(n, 11 * step + i * 0x9E3779B9)
            ref[i] = (*moment_codes(m1, um, 2), *moment_codes(v1, uv, 4))
            for got, exp in zip((mm[i].codes, mm[i].scale, vv[i].codes, vv[i].scale), ref[i]):
                np.testing.assert_array_equal(got.cpu().numpy(), exp, err_msg=f"step {step} tensor {i}")
            up = formula(before[i], g[i], torch.from_numpy(m0).cuda(), torch.from_numpy(v0).cuda(), step)[3]
            check_p(p[i], torch.from_numpy(want).cuda(), up, before[i], dtype)
    first, second = sft.moment_values(mm, "first"), sft.moment_values(vv, "second")
    for i in range(len(SIZES)):
        np.testing.assert_array_equal(first[i].cpu().numpy(), moment_values(*ref[i][:2], 2))
        np.testing.assert_array_equal(second[i].cpu().numpy(), moment_values(*ref[i][2:], 4))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_sf8_not_finite_shows_in_its_block_only(gpu, bad):
    n = 5 * BLOCK + 9
    p, g, _, _ = make([n], torch.float32)
    g[0][2 * BLOCK + 5] = bad
    m, v = [sft.SF8Moment.zeros(n, "cuda")], [sft.SF8Moment.zeros(n, "cuda")]
    for step in (1, 2):
        sft.adamw_step(p, g, m, v, step=step, **HYPER)
    hit = torch.zeros(n, dtype=torch.bool, device="cuda")
    hit[2 * BLOCK:3 * BLOCK] = True
    for val in (sft.moment_values(m, "first")[0], sft.moment_values(v, "second")[0]):
        assert torch.equal(val.isnan(), hit)
    assert bool(p[0][~hit].isfinite().all()) and bool(p[0][2 * BLOCK + 5].isnan())


def test_f32_not_finite_stays_in_its_element(gpu):
    p, g, m, v = make([1000], torch.float32)
    g[0][17] = float("nan")
    sft.adamw_step(p, g, m, v, step=1, **HYPER)
    for t in (p[0], m[0], v[0]):
        assert t.isnan().nonzero().flatten().tolist() == [17]


@pytest.mark.parametrize("state", ["f32", "sf8"])
@pytest.mark.parametrize("dtype", TYPES)
def test_views_that_are_not_aligned(gpu, dtype, state):
    """Parameters and gradients at odd offsets of a wider buffer: the same bits as aligned copies, and the
    elements around them untouched."""
    n = 3001
    p, g, m, v = make([n], dtype)
    mom = lambda: ([m[0].clone()], [v[0].clone()]) if state == "f32" else (  # noqa: E731
        [sft.SF8Moment.zeros(n, "cuda")], [sft.SF8Moment.zeros(n, "cuda")])
    want = p[0].clone()
    m1, v1 = mom()
    sft.adamw_step([want], g, m1, v1, step=2, **HYPER)
    for off in (1, 2, 3):
        wide, gw = torch.full((n + 9,), 7.0, dtype=dtype, device="cuda"), torch.zeros(n + 9, dtype=dtype, device="cuda")
        wide[off:off + n] = p[0]
        gw[off + 1:off + 1 + n] = g[0]
        m2, v2 = mom()
        sft.adamw_step([wide[off:off + n]], [gw[off + 1:off + 1 + n]], m2, v2, step=2, **HYPER)
        assert torch.equal(wide[off:off + n], want)
        assert bool((wide[:off] == 7).all()) and bool((wide[off + n:] == 7).all())
        for a, b in zip(m1 + v1, m2 + v2):
            if state == "sf8":
                assert torch.equal(a.codes, b.codes) and torch.equal(a.scale, b.scale)
            else:
                assert torch.equal(a, b)


def test_layouts(gpu):
    """A transposed parameter, and a gradient of another layout (copied)."""
    p = torch.randn(40, 30, device="cuda", generator=gen()).t()
    g = torch.randn(30, 40, device="cuda", generator=gen(1))
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    assert p.stride() == m.stride() != g.stride()
    want = formula(p, g, m, v, 1)
    before = p.clone()
    sft.adamw_step([p], [g], [m], [v], step=1, **HYPER)
    check_p(p, want[0], want[3], before, torch.float32)
    gap = torch.zeros(8, 8, device="cuda")[:, :5]
    with pytest.raises(SFShapeError, match="gaps"):
        sft.adamw_step([gap], [torch.zeros_like(gap)], [torch.zeros_like(gap)], [torch.zeros_like(gap)], step=1, lr=1.0)


def test_many_tensors(gpu):
    """More tensors than one launch's table holds, empty ones among them."""
    sizes = [(i * 37) % 300 for i in range(1000)]
    p, g, m, v = make(sizes, torch.float32)
    old = [[t.clone() for t in x] for x in (p, g, m, v)]
    sft.adamw_step(p, g, m, v, step=1, **HYPER)
    cat = lambda x: torch.cat(list(x))  # noqa: E731
    want, m1, _, up = formula(*(cat(x) for x in old), 1)
    check_p(cat(p), want, up, cat(old[0]), torch.float32)
    assert bool(((cat(m).double() - m1).abs() <= 1e-8).all())


def test_mixed_types_and_kinds_in_one_call(gpu):
    sizes, kinds = [300, 5000, 700, 6000], [0, 1, 1, 0]
    p, g, m, v = [], [], [], []
    for i, (n, k) in enumerate(zip(sizes, kinds)):
        a, b, c, d = make([n], TYPES[i % 3], i)
        p, g = p + a, g + b
        m += [sft.SF8Moment.zeros(n, "cuda")] if k else c
        v += [sft.SF8Moment.zeros(n, "cuda")] if k else d
    m0, v0 = sft.moment_values(m, "first"), sft.moment_values(v, "second")
    old = [[t.clone() for t in x] for x in (p, g, m0, v0)]
    sft.adamw_step(p, g, m, v, step=4, **HYPER)
    for i in range(4):
        want, _, _, up = formula(*(x[i] for x in old), 4)
        check_p(p[i], want, up, old[0][i], p[i].dtype)


def test_the_same_tensor_twice_is_refused(gpu):
    p, g, m, v = make([500, 500], torch.float32)
    before = p[0].clone()
    for args in (([p[0]] * 2, g, m, v), (p, g, [m[0]] * 2, v), ([p[0], p[0][100:400]], [g[0], g[1][:300]], [m[0], m[1][:300]],
                                                               [v[0], v[1][:300]]), (p, [p[0], g[1]], m, v)):
        with pytest.raises(SFShapeError, match="given twice"):
            sft.adamw_step(*args, step=1, lr=1.0)
    assert torch.equal(p[0], before)
    shared = [g[0], g[0]]                                             # a gradient may be shared: it is only read
    sft.adamw_step(p, shared, m, v, step=1, **HYPER)


def test_moment_refusals(gpu):
    p, g, m, v = make([500], torch.float32)
    z = sft.SF8Moment.zeros(500, "cuda")
    with pytest.raises(SFTypeError, match="one moment in sf8"):
        sft.adamw_step(p, g, [z], v, step=1, lr=1.0)
    with pytest.raises(SFTypeError, match="float16"):
        sft.adamw_step(p, g, [m[0].half()], v, step=1, lr=1.0)
    with pytest.raises(SFShapeError, match="another shape"):
        sft.adamw_step(p, g, [m[0][:499]], v, step=1, lr=1.0)
    for wrong in (sft.SF8Moment(z.codes[:499], z.scale), sft.SF8Moment(z.codes, z.scale[:1]),
                  sft.SF8Moment(z.codes.cpu(), z.scale),
                  sft.SF8Moment(torch.zeros(1000, dtype=torch.int8, device="cuda")[::2], z.scale),
                  sft.SF8Moment(torch.zeros(504, dtype=torch.int8, device="cuda")[1:501], z.scale)):
        with pytest.raises(SFShapeError):
            sft.adamw_step(p, g, [wrong], [z], step=1, lr=1.0)
    with pytest.raises(SFTypeError, match="int8"):
        sft.adamw_step(p, g, [sft.SF8Moment(z.codes.float(), z.scale)], [z], step=1, lr=1.0)


def test_another_stream(gpu):
    p, g, m, v = make([100000], torch.float32)
    want = [t.clone() for t in p]
    sft.adamw_step(want, g, [m[0].clone()], [v[0].clone()], step=1, **HYPER)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sft.adamw_step(p, g, m, v, step=1, **HYPER)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(p[0], want[0])


def model(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(96, 80), torch.nn.GELU(), torch.nn.Linear(80, 96)).cuda().to(dtype)


def backward(net, i):
    x = torch.randn(16, 96, device="cuda", generator=gen(100 + i)).to(next(net.parameters()).dtype)
    net.zero_grad()
    (net(x).float() - x.float()).square().mean().backward()


@pytest.mark.parametrize("state", ["float32", "sf8"])
def test_optimizer_against_torch(gpu, state):
    """Five steps beside torch.optim.AdamW on the same gradients.  float32: the parameters differ by roundings,
    under 5 steps x 2^-20 of an update of at most lr x sqrt(1 / (1 - b2)) and 5 x 2 x 2^-24 of the value.  sf8: the
    updates differ by the rounding of the moments; the moments of the last step must be the step's own."""
    net = model()
    ref = [p.detach().clone().requires_grad_() for p in net.parameters()]
    opt, want = sft.AdamW(net.parameters(), state=state, **HYPER), torch.optim.AdamW(ref, **HYPER)
    for i in range(5):
        backward(net, i)
        for p, r in zip(net.parameters(), ref):
            r.grad = p.grad.clone()
        opt.step()
        want.step()
    for p, r in zip(net.parameters(), ref):
        assert opt.steps_done(p) == 5
        m, v = opt.moments(p)
        assert m.shape == p.shape and v.shape == p.shape
        big = HYPER["lr"] * (1 - HYPER["betas"][1]) ** -0.5
        if state == "float32" or p.numel() < 4096:
            assert float((p - r).abs().max()) <= 5 * (2.0 ** -20 * big + 2 * 2.0 ** -24 * float(r.detach().abs().max()))
        else:
            assert opt.state[p]["exp_avg"].dtype == torch.int8
            assert float((p - r).abs().max()) <= 5 * 2 * big


def test_groups_missing_gradients_and_late_ones(gpu):
    a, b = (torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2))
    opt = sft.AdamW([{"params": [a], "lr": 0.5}, {"params": [b], "weight_decay": 0.0}], lr=0.1)
    a.grad = torch.ones_like(a)
    opt.step()
    assert float(b[0]) == 1.0 and opt.steps_done(b) == 0
    b.grad = torch.ones_like(b)
    opt.step()
    assert opt.steps_done(a) == 2 and opt.steps_done(b) == 1
    # the first step moves by lr (1 - eps / (1 + eps)): bias corrections cancel the moments' decays
    assert abs(float(b[0]) - 0.9) < 1e-6


@pytest.mark.parametrize("state", ["float32", "sf8"])
def test_state_dict_round_trip(gpu, state):
    """Saved after two steps and loaded into a new optimizer, the third step gives the same bits."""
    nets = [model(torch.bfloat16) for _ in range(2)]
    opts = [sft.AdamW(n.parameters(), state=state, **HYPER) for n in nets]
    for i in range(2):
        backward(nets[0], i)
        opts[0].step()
    nets[1].load_state_dict(nets[0].state_dict())
    saved = opts[0].state_dict()
    opts[1].load_state_dict(saved)
    for k, st in opts[1].state.items():
        for name, t in st.items():
            if isinstance(t, torch.Tensor):
                assert t.dtype in ((torch.int8, torch.float32) if state == "sf8" else (torch.float32,))
    for net, opt in zip(nets, opts):
        backward(net, 2)
        opt.step()
    for p, q in zip(nets[0].parameters(), nets[1].parameters()):
        assert torch.equal(p, q) and opts[1].steps_done(q) == 3


@pytest.mark.parametrize("state", ["float32", "sf8"])
def test_captured_steps_equal_eager_ones(gpu, state):
    """A captured step replayed gives what eager steps give: the count and the dither advance on the device."""
    nets = [model() for _ in range(2)]
    opts = [sft.AdamW(n.parameters(), state=state, capturable=True, **HYPER) for n in nets]
    for net, opt in zip(nets, opts):
        backward(net, 0)
        opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for _ in range(4):
        graph.replay()
        opts[1].step()
    torch.cuda.synchronize()
    for p, q in zip(nets[0].parameters(), nets[1].parameters()):
        assert torch.equal(p, q)
        assert opts[0].steps_done(p) == 5
    assert opts[0].state_dict()["state"][0]["step"] == 5


def test_capturable_equals_host_steps(gpu):
    """The constants of the device counter are the host's (both from float64 powers; one unit of float32 apart)."""
    nets = [model() for _ in range(2)]
    opts = [sft.AdamW(n.parameters(), capturable=c, **HYPER) for n, c in zip(nets, (True, False))]
    for i in range(3):
        for net, opt in zip(nets, opts):
            backward(net, i) if i == 0 else None
            opt.step()
    for p, q in zip(nets[0].parameters(), nets[1].parameters()):
        assert float((p - q).abs().max()) <= 3 * (2.0 ** -22 * HYPER["lr"] * 10 + 2.0 ** -23 * float(q.abs().max()))


def test_capture_refusals(gpu):
    net = model()
    backward(net, 0)
    plain, late = sft.AdamW(net.parameters()), sft.AdamW(net.parameters(), capturable=True)
    plain.step()
    for opt, what in ((plain, "capturable=True"), (late, "before the capture")):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(SFUnsupportedError, match=what):
            with torch.cuda.graph(graph):
                opt.step()
    late.step()
    next(net.parameters()).grad = None
    with pytest.raises(SFUnsupportedError, match="needs its gradient"):
        late.step()


@pytest.mark.parametrize("state", ["float32", "sf8"])
def test_a_step_is_seen_by_the_layers_that_keep_codes_and_by_autograd(state):
    """A chain layer keeps its weight's codes until the weight changes; autograd refuses a parameter that changed
    between its use and the backward pass."""
    torch.manual_seed(0)
    net = sft.convert(torch.nn.Sequential(torch.nn.Linear(128, 64)).cuda(), dtype="sf16")
    x = torch.randn(4, 128, generator=gen(), device="cuda") * 0.1
    with torch.no_grad():
        before = net(x)
    opt = sft.AdamW(net.parameters(), lr=0.05, state=state)
    net(x).sum().backward()
    opt.step()
    fresh = sft.convert(torch.nn.Sequential(torch.nn.Linear(128, 64)).cuda(), dtype="sf16")
    fresh.load_state_dict(net.state_dict())
    with torch.no_grad():
        after, want = net(x), fresh(x)
    assert torch.equal(after, want) and not torch.equal(after, before)
    w = net[0].weight
    y = (w * w).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_step_on_inference_tensors():
    with torch.inference_mode():
        p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
        m, v = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
        sft.adamw_step([p], [g], [m], [v], step=1, lr=0.5)
    # a first step moves by lr times g / |g|
    assert float((p - 0.5).abs().max()) < 1e-6


def test_a_parameter_twice_with_moments_of_two_kinds_is_refused_before_anything_runs():
    p, g, m, v = make([5000], torch.float32)
    before, z = p[0].clone(), [sft.SF8Moment.zeros(5000, "cuda") for _ in range(2)]
    with pytest.raises(SFShapeError, match="given twice"):
        sft.adamw_step(p * 2, g * 2, [m[0], z[0]], [v[0], z[1]], step=1, lr=1.0)
    assert torch.equal(p[0], before)
    empty = torch.empty(0, device="cuda")                    # no elements, no place in memory
    sft.adamw_step([empty, empty], [empty, empty], [empty, empty], [empty, empty], step=1, lr=1.0)


@pytest.mark.parametrize("mode", ["chain", "wide"])
def test_replayed_steps_and_the_codes_that_layers_keep(mode):
    """A replay does not count in the parameters' versions: the layers' codes are cleared by hand."""
    torch.manual_seed(0)
    make_net = lambda: sft.convert(torch.nn.Sequential(torch.nn.Linear(128, 64)).cuda(), dtype="sf16",  # noqa: E731
                                   accumulate=mode, attention=False)
    net, x = make_net(), torch.randn(4, 128, generator=gen(), device="cuda") * 0.1
    opt = sft.AdamW(net.parameters(), lr=0.05, capturable=True)
    for p in net.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    with torch.no_grad():
        before = net(x)
        graph.replay()
        sft.weight_cache.clear()
        sft.wide_weight_cache.clear()
        after = net(x)
        fresh = make_net()
        fresh.load_state_dict(net.state_dict())
        assert torch.equal(after, fresh(x)) and not torch.equal(after, before)
