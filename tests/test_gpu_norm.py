"""Layer norm on the B200 against its formula in 64 bits.

Tolerances, with u = 2^-24 (half a step of float32) and e = finfo(type).eps; a sum over a row has at most 64 roundings
in its longest chain (32 elements a lane, 5 exchanges, 16 warps, 8 CTAs):

* the mean is off by dm = 65 u mean|x|, a deviation by dm + u |x - mean|;
* the variance, relative: 2 dm r + 70 u; so r is off by dm r + 35 u + 2^-22 (rsqrt is two steps off at most), relative;
* xh by dm r (1 + |xh|) + 45 u |xh|;
* y by |w| times that and 2 u (|w xh| + |y|), and half a step of its type;
* the backward pass's means by 70 u of the mean of the magnitudes, and by what xh is off; dx by these and 6 u of each
  of its three terms and by what r is off;
* dw and db: at most M / 18 + 100 roundings of a column's sum (rows of a team, teams joined), u of the magnitudes each.
"""
import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200._errors import SFShapeError, SFTypeError, SFUnsupportedError

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24
# rows and features: one of each, a warp's row and its borders, a CTA's, clusters of 2 to 8 CTAs
SIZES = [(1, 1), (3, 2), (5, 7), (64, 8), (130, 31), (33, 256), (7, 257), (20, 768), (9, 1000), (6, 1024), (5, 1025), (301, 1031),
         (4, 2049), (12, 4096), (3, 8192), (2, 8193), (3, 16384), (2, 40001), (2, 65536), (5000, 16), (1, 768)]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * std).to(dtype)


def formula(x, w, b, dy=None, eps=1e-5):
    """[(value, tolerance before the result's rounding)] of y and, with dy, of dx, dw and db."""
    x, D = x.detach().double(), x.shape[-1]
    w = torch.ones(D, device="cuda").double() if w is None else w.detach().double()
    b = torch.zeros(D, device="cuda").double() if b is None else b.detach().double()
    mean = x.mean(1, keepdim=True)
    r = ((x - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * r
    dm = 65 * U * x.abs().mean(1, keepdim=True)
    rel = dm * r + 35 * U + 2.0 ** -22
    off = dm * r * (1 + xh.abs()) + (45 * U + 2.0 ** -22) * xh.abs()
    y = xh * w + b
    out = [(y, w.abs() * off + 2 * U * ((xh * w).abs() + y.abs()))]
    if dy is None:
        return out
    dy = dy.double()
    gy = dy * w
    a, c = gy.mean(1, keepdim=True), (gy * xh).mean(1, keepdim=True)
    da = 70 * U * gy.abs().mean(1, keepdim=True)
    dc = 70 * U * (gy * xh).abs().mean(1, keepdim=True) + (gy.abs() * off).mean(1, keepdim=True)
    dx = r * (gy - a - xh * c)
    tol = r * (da + xh.abs() * dc + c.abs() * off + 6 * U * (gy.abs() + a.abs() + (xh * c).abs())) + dx.abs() * rel
    n = x.shape[0] // 18 + 100
    out.append((dx, tol))
    out.append(((dy * xh).sum(0), n * U * (dy * xh).abs().sum(0) + (dy.abs() * off).sum(0)))
    out.append((dy.sum(0), n * U * dy.abs().sum(0)))
    return out


def close(got, want, tol):
    info = torch.finfo(got.dtype)
    bound = tol * (1 + info.eps) + info.eps / 2 * want.abs() + info.tiny * info.eps
    assert got.shape == want.shape
    ratio = ((got.detach().double() - want).abs() / bound).max() if got.numel() else torch.zeros(())
    assert float(ratio) <= 1, float(ratio)


def run(x, w, b, dy, **kw):
    wanted = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = sft.layer_norm(x, w, b, **kw)
    return [y.detach(), *torch.autograd.grad(y, wanted, dy)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,d", SIZES)
def test_values_and_gradients(gpu, m, d, dtype):
    for i, params in enumerate([dtype, torch.float32]):
        x = randn(m, d, seed=i, dtype=dtype) + (3 if i else 0)
        w, b = (1 + randn(d, seed=2, std=0.3)).to(params), randn(d, seed=3, dtype=params)
        if i and d % 2:
            b = None
        dy = randn(m, d, seed=4, dtype=dtype)
        want = formula(x, w, b, dy)
        got = run(x, w, b, dy)
        assert got[0].dtype == dtype and got[1].dtype == dtype and got[2].dtype == params
        for g, (v, t) in zip(got, want):
            close(g, v, t)
        with torch.no_grad():
            assert torch.equal(sft.layer_norm(x, w, b), got[0])
            close(sft.layer_norm(x, None, b), *formula(x, None, b)[0])
        gx, = torch.autograd.grad(sft.layer_norm(x), x, dy)
        close(gx, *formula(x, None, None, dy)[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [40, 1031, 2048])
def test_layouts(gpu, d, dtype):
    """Rows of a wider buffer at any offset, transposed and broadcast rows, strided parameters: the formula's values."""
    x, dy = randn(6, 5, d, seed=1, dtype=dtype), randn(6, 5, d, seed=2, dtype=dtype)
    w, b = randn(d, seed=3, dtype=dtype), randn(d, seed=4, dtype=dtype)
    want = [(v.view(6, 5, d) if v.dim() == 2 else v, t.view(6, 5, d) if t.dim() == 2 else t)
            for v, t in formula(x.view(-1, d), w, b, dy.view(-1, d))]
    for off in (0, 1, 8):
        xs = torch.zeros(6, 5, d + 16, dtype=dtype, device="cuda")[..., off:off + d].copy_(x)
        gs = torch.zeros(6, 5, d + 9, dtype=dtype, device="cuda")[..., 9 - off:d + 9 - off].copy_(dy)
        for g, (v, t) in zip(run(xs, w, b, gs), want):
            close(g, v, t)
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    gt = dy.transpose(0, 2).contiguous().transpose(0, 2)
    ws = torch.zeros(2 * d, dtype=dtype, device="cuda")[::2].copy_(w)
    wo = torch.zeros(d + 1, dtype=dtype, device="cuda")[1:].copy_(w)
    for ww in (ws, wo):
        for g, (v, t) in zip(run(xt, ww, b, gt), want):
            close(g, v, t)
    row = randn(d, seed=5, dtype=dtype)
    y = sft.layer_norm(row.expand(4, 3, d), w, b)
    assert torch.equal(y, sft.layer_norm(row, w, b).expand(4, 3, d))
    assert sft.layer_norm(x[0, 0], w, b).shape == (d,)


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_batches(gpu, dtype):
    x = torch.zeros(2, 0, 24, dtype=dtype, device="cuda")
    y, gx, gw, gb = run(x, randn(24), randn(24), x.clone())
    assert y.shape == x.shape and gx.shape == x.shape and not bool(gw.any()) and not bool(gb.any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 1500])
def test_rows_that_are_constant_far_or_not_finite(gpu, d, dtype):
    """A constant row has no deviation; a row far from zero keeps its own; NaN and infinity stay in their rows."""
    x = randn(40, d, dtype=dtype)
    x[1] = 5.0
    x[2] += 1000
    x[3] = 0
    want, tol = formula(x, None, None)[0]
    y = sft.layer_norm(x)
    close(y, want, tol)
    assert not bool(y[1].any()) and not bool(y[3].any())
    x[7, 3], x[9, 0] = float("nan"), float("inf")
    z = sft.layer_norm(x)
    hit = torch.zeros(40, dtype=torch.bool, device="cuda")
    hit[7] = hit[9] = True
    assert bool(z[hit].isnan().all()) and torch.equal(z[~hit], y[~hit])


def test_against_differences(gpu):
    """The gradients of float32 inputs against differences of the formula in 64 bits."""
    x, w, b, dy = randn(5, 37), 1 + randn(37, seed=1), randn(37, seed=2), randn(5, 37, seed=3)
    got = run(x, w, b, dy)[1:]
    x, w, b = (t.detach().double() for t in (x, w, b))

    def loss():
        return (formula(x, w, b)[0][0] * dy.double()).sum()

    for t, g in zip((x, w, b), got):
        for i in range(0, t.numel(), 7):
            flat, h = t.view(-1), 1e-4
            at = float(flat[i])
            flat[i] = at + h
            up = loss()
            flat[i] = at - h
            down = loss()
            flat[i] = at
            # (a third difference over 6, below 1e2 h^2 here, and float32's own part)
            assert abs(float((up - down) / (2 * h)) - float(g.reshape(-1)[i])) < 1e-5 * (1 + abs(float(g.reshape(-1)[i])))


def test_single_gradients(gpu):
    """Each gradient alone is the one that all together give."""
    x, w, b, dy = randn(50, 300, dtype=torch.bfloat16), randn(300, seed=1), randn(300, seed=2), randn(50, 300, seed=3).bfloat16()
    whole = run(x, w, b, dy)[1:]
    for i in range(3):
        one = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        g, = torch.autograd.grad(sft.layer_norm(*one), one[i], dy)
        assert torch.equal(g, whole[i])


def test_the_same_bits_each_time_and_streams(gpu):
    x, w, b, dy = randn(3000, 768, dtype=torch.bfloat16), randn(768, seed=1), randn(768, seed=2), randn(3000, 768, seed=3).bfloat16()
    first = run(x, w, b, dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run(x, w, b, dy))
    torch.cuda.synchronize()
    for other in got:
        assert all(torch.equal(a, c) for a, c in zip(first, other))


def test_captured(gpu):
    """Forward and backward in one graph, replayed on new values."""
    w, b = randn(1000, seed=1).requires_grad_(), randn(1000, seed=2).requires_grad_()
    x = randn(70, 1000, dtype=torch.float16).requires_grad_()
    dy = randn(70, 1000, seed=3, dtype=torch.float16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = sft.layer_norm(x, w, b)
        torch.autograd.grad(y, (x, w, b), dy)
        del y
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = sft.layer_norm(x, w, b)
        grads = torch.autograd.grad(y, (x, w, b), dy)
    for seed in (7, 8):
        with torch.no_grad():
            x.copy_(randn(70, 1000, seed=seed, dtype=torch.float16))
            dy.copy_(randn(70, 1000, seed=seed + 9, dtype=torch.float16))
        graph.replay()
        for g, want in zip([y.detach(), *grads], run(x.detach().clone(), w.detach(), b.detach(), dy)):
            assert torch.equal(g, want)


def test_kept_tensors_on_the_host(gpu):
    x, w, b, dy = randn(20, 130, dtype=torch.bfloat16), randn(130, seed=1), randn(130, seed=2), randn(20, 130, seed=3).bfloat16()
    xs = torch.zeros(20, 200, dtype=torch.bfloat16, device="cuda")[:, 3:133].copy_(x)
    want = run(x, w, b, dy)
    with torch.autograd.graph.save_on_cpu():
        got = run(xs, w, b, dy)
    for a, c, (v, t) in zip(got, want, formula(x, w, b, dy)):
        close(a, v, t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,d", [(900, 8200), (700, 8201), (500, 16384), (500, 20001), (300, 65536), (150, 40001)])
def test_long_rows_in_turn(gpu, m, d, dtype):
    """Clusters that take rows one after another, and the same in two streams at once and in a replayed graph.
    (A column's sum: 300 rows of 16 clusters are 19 to a cluster and 16 to be joined, of the 116 that are allowed.)"""
    x, w, b = randn(m, d, seed=1, dtype=dtype) + 1, 1 + randn(d, seed=2, std=0.3), randn(d, seed=3)
    dy = randn(m, d, seed=4, dtype=dtype)
    got = run(x, w, b, dy)
    for g, (v, t) in zip(got, formula(x, w, b, dy)):
        close(g, v, t)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    again = []
    for s in streams:
        with torch.cuda.stream(s):
            again.append(run(x, w, b, dy))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = sft.layer_norm(x, w, b)
    graph.replay()
    assert torch.equal(y, got[0])
    for other in again:
        assert all(torch.equal(g, o) for g, o in zip(got, other))


def test_a_wait_that_runs_out_is_reported(gpu):
    """Parts of a long row that never come: the rows are NaN, it is counted, and the next call is as if nothing had been."""
    from superfloat.python_b200 import _lib
    x = randn(7, 20000)
    want, before = sft.layer_norm(x), sft.tensor_failures()
    _lib.load().sfb_wide_wait_limit(2000, 1)
    try:
        y = sft.layer_norm(x)
    finally:
        _lib.load().sfb_wide_wait_limit(0, 0)
    assert bool(y.isnan().all()) and sft.tensor_failures() > before
    assert torch.equal(sft.layer_norm(x), want)


def test_refusals(gpu):
    x, w = randn(4, 8), randn(8)
    with pytest.raises(SFTypeError):
        sft.layer_norm(x.double())
    with pytest.raises(SFShapeError):
        sft.layer_norm(x, randn(7))
    with pytest.raises(SFTypeError):
        sft.layer_norm(x, w.double())
    with pytest.raises(SFShapeError):
        sft.layer_norm(x, w.cpu())
    with pytest.raises(SFShapeError):
        sft.layer_norm(torch.zeros(2, 65537, device="cuda"))
    with pytest.raises(ValueError):
        sft.layer_norm(x, w, eps=-1.0)
    y = sft.layer_norm(x.requires_grad_(), w)
    g, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    import torch.autograd.forward_ad as fa
    with fa.dual_level(), pytest.raises(SFUnsupportedError):
        sft.layer_norm(fa.make_dual(x.detach(), x.detach()), w)
