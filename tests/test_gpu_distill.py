"""The distillation loss on the B200 against its formula in 64 bits.

Tolerances, with u = 2^-24 and z = (x - max) / T: an exponential's argument is off by 3 u |z| (a difference, the
factor and their product), the exponential itself by 2^-22 of its value; a row's sum has at most n = 2 (V / 4096 + 70)
additions and changes of the maximum in its longest chain, each off by at most 2^-22.  So q, p and their sums are off by
rel = 3 u |z| + 3 u mean|z| + n 2^-22, relative, and a logarithm by that and u of its value; a row's loss by rel of
sum p (|log p| + |log q| + 3), and 64 u of it for the sum; the sum of M rows by (M / 1024 + 40) u.
The gradient is off by (q + p) rel of the row's factor, and half a step of its type.
"""
import math

import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200._errors import SFShapeError, SFTypeError, SFUnsupportedError

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24
# rows, vocabulary, entries: a vocabulary of one, odd ones, clusters of 1 to 8 CTAs, parts that shared memory does not hold
SIZES = [(1, 1, 1), (2, 3, 5), (3, 7, 2), (5, 8, 8), (40, 257, 16), (13, 1000, 1), (7, 4097, 33), (3, 8200, 64), (300, 1031, 7), (2, 50257, 64),
         (350, 50257, 3), (1, 120001, 200), (4, 600, 600), (2, 900, 1024), (900, 33, 4)]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * std).to(dtype)


def entries(m, v, k, seed=0, t_dtype=torch.float32, absent=True):
    """Teacher's logits in falling order with random places, doubles among them; every third row ragged, one in five empty."""
    t = randn(m, k, seed=seed, std=3).sort(1, descending=True).values.to(t_dtype)
    i = torch.randint(0, v, (m, k), generator=gen(seed + 1), device="cuda")
    if absent:
        i[::3, k - k // 3:] = -1
        i[4::5] = -1
    return t, i


def rows64(logits, t, i, T, n_sum=None):
    """(loss, its tolerance, gradient for a factor of one, its tolerance) of every row; rows without entries are 0."""
    x = logits.detach().double() / T
    V = x.shape[-1]
    there = (i >= 0) & (i < V) & (t.double() != -math.inf)
    t = torch.where(there, t.double() / T, torch.full_like(t, -math.inf, dtype=torch.double))
    some = there.any(1)
    t = torch.where(some[:, None], t, torch.zeros_like(t))
    logp = torch.log_softmax(t, 1)
    p = logp.exp() * there
    z = x - x.amax(1, keepdim=True)
    logq = torch.log_softmax(x, 1)
    q = logq.exp()
    at = i.clamp(0, V - 1).long()
    lq = logq.gather(1, at)
    row = torch.where(p > 0, p * (logp - lq), torch.zeros_like(p)).sum(1) * T * T
    zq = torch.where(q > 0, z.abs() * q, torch.zeros_like(q)).sum(1, keepdim=True)
    tz = torch.where(p > 0, (t - t.amax(1, keepdim=True)).abs(), torch.zeros_like(p)).amax(1, keepdim=True)
    rel = lambda a: 3 * U * (a + zq + 2 * tz) + 2 * (V / 4096 + 70) * 2.0 ** -22  # noqa: E731
    lp = torch.where(p > 0, logp.abs(), torch.zeros_like(p))
    weight = torch.where(p > 0, p * (lp + lq.abs() + 3) * (rel(z.gather(1, at).abs()) + 64 * U), torch.zeros_like(p))
    mass = torch.zeros_like(x).scatter_add(1, at, p)
    grad = T * (q - mass)
    tol = T * (q * rel(z.abs().clamp(max=1e4)) + mass * rel(torch.zeros_like(z)))
    row, weight = row * some, weight.sum(1) * T * T * some
    return row, weight, grad * some[:, None], tol * some[:, None], some


def close(got, want, tol, dtype=None):
    info = torch.finfo(got.dtype)
    bound = tol * (1 + info.eps) + info.eps / 2 * want.abs() + info.tiny * info.eps + 2.0 ** -126
    assert got.shape == want.shape
    ratio = ((got.detach().double() - want).abs() / bound).max() if got.numel() else torch.zeros(())
    assert float(ratio) <= 1, float(ratio)


def reduced(row, tol, some, w, reduction):
    """(loss, tolerance, each row's factor)."""
    w = torch.ones_like(row) if w is None else w.double()
    w = torch.where(some, w, torch.zeros_like(w))
    row, tol = torch.where(w != 0, row * w, torch.zeros_like(row)), torch.where(w != 0, tol * w.abs(), torch.zeros_like(row))
    n = (row.numel() / 1024 + 40) * U
    if reduction == "none":
        return row, tol + 4 * U * row.abs(), w
    share = torch.ones((), device="cuda").double()
    if reduction == "mean":
        share = torch.where(w.sum() == 0, torch.zeros_like(share), 1 / w.sum())
    return row.sum() * share, (tol.sum() + n * row.abs().sum() + 4 * U * row.abs().sum()) * share.abs() * (1 + n), w * share


def check(logits, t, i, T=1.0, w=None, reduction="mean", g=None):
    row, tol, grad, gtol, some = rows64(logits.detach().reshape(-1, logits.shape[-1]), t.reshape(-1, t.shape[-1]),
                                        i.reshape(-1, i.shape[-1]), T)
    flat = None if w is None else w.reshape(-1)
    loss, tol, factor = reduced(row, tol, some, flat, reduction)
    x = logits.detach().requires_grad_()
    got = sft.distill_loss(x, t, i, temperature=T, row_weight=w, reduction=reduction)
    assert got.dtype == torch.float32 and got.shape == (logits.shape[:-1] if reduction == "none" else ())
    close(got.reshape(-1), loss.reshape(-1), tol.reshape(-1))
    with torch.no_grad():
        assert torch.equal(sft.distill_loss(x, t, i, temperature=T, row_weight=w, reduction=reduction), got)
    g = torch.ones_like(got) if g is None else g
    gx, = torch.autograd.grad(got, x, g)
    assert gx.shape == logits.shape and gx.dtype == logits.dtype
    factor = (factor * g.double().reshape(-1)).nan_to_num()[:, None]
    kept = factor != 0
    zero = torch.zeros_like(grad)
    want = torch.where(kept, grad * factor, zero)
    # (the mean's denominator is a sum of M weights, and the factor four products)
    n = row.numel() / 256 + 20
    off = torch.where(kept, (gtol + n * U * grad.abs()) * factor.abs(), zero)
    close(gx.reshape(-1, logits.shape[-1]), want, off)
    return got, gx


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,v,k", SIZES)
def test_values_and_gradients(gpu, m, v, k, dtype):
    logits = randn(m, v, seed=1, dtype=dtype, std=3)
    t, i = entries(m, v, k, seed=2, t_dtype=dtype)
    check(logits, t, i)
    check(logits, t, i.int(), T=2.5, reduction="sum", g=torch.tensor(-3.0, device="cuda"))
    w = randn(m, seed=3).abs() * (randn(m, seed=4) > -0.5)
    check(logits, t, i, T=0.5, w=w, reduction="none", g=randn(m, seed=5))
    check(logits, t.float(), i, w=randn(m, seed=4) > 0, g=torch.tensor(0.25, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(gpu, dtype):
    """Rows of a wider buffer, all but the last row of each sequence, transposed and broadcast rows, odd offsets."""
    B, S, v, k = 3, 7, 515, 9
    t, i = entries(B * S, v, k, seed=2)
    t, i = t.view(B, S, k), i.view(B, S, k)
    w = (randn(B, S, seed=3) > -1)
    x = randn(B, S, v, seed=1, dtype=dtype, std=2)
    want = check(x, t, i, w=w)
    for off in (0, 1, 2, 8):
        wide = torch.zeros(B, S, v + 9, dtype=dtype, device="cuda")[..., off:off + v].copy_(x)
        far = torch.zeros(B, S, 2 * v + 9, dtype=dtype, device="cuda")[..., off:off + v].copy_(x)
        for xs in (wide, far):                        # (where a row starts within 16 bytes sets the order of its sum)
            check(xs, t, i, w=w)
    longer = torch.zeros(B, S + 1, v, dtype=dtype, device="cuda")
    longer[:, :-1] = x
    for xs in (longer[:, :-1], x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(0, 2).contiguous().transpose(0, 2)):
        check(xs, t, i, w=w)
    check(x[:1, :1].expand(B, S, v), t, i, w=w)
    ts = torch.zeros(B, S, 2 * k, device="cuda")[..., ::2].copy_(t)
    js = torch.zeros(B, S, k + 3, device="cuda", dtype=torch.int64)[..., 3:].copy_(i)
    ws = torch.zeros(S, B, device="cuda", dtype=torch.bool).t().copy_(w)
    got = check(x, ts, js, w=ws)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = check(x[0, 0], t[0, 0], i[0, 0], reduction="none")
    assert one[0].shape == ()


@pytest.mark.parametrize("dtype", TYPES)
def test_entries_that_are_absent_doubled_or_out_of_range(gpu, dtype):
    v = 100
    x = randn(6, v, dtype=dtype)
    t = randn(6, 5, seed=1)
    i = torch.tensor([[1, 2, 3, 4, 5], [7, 7, 7, 7, 7], [-1, 3, v, -9, 2 ** 40], [-1] * 5, [0, v - 1, 0, v - 1, 50], [9, 8, 7, 6, 5]], device="cuda")
    t[4, 2] = t[5, :] = -math.inf
    for reduction in ("mean", "sum", "none"):
        loss, g = check(x, t, i, reduction=reduction)
        assert not bool(g[3].any()) and not bool(g[5].any())
    check(x, t.to(torch.float16), i.clamp(-2 ** 31, 2 ** 31 - 1).int())


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_rows_hide_what_they_hold(gpu, dtype):
    """NaN and infinities in rows of weight 0 or without entries change nothing; elsewhere they show in their row."""
    x, (t, i) = randn(8, 300, dtype=dtype), entries(8, 300, 6, absent=False)
    w = torch.ones(8, device="cuda")
    w[2] = 0
    i[5] = -1
    want = check(x, t, i, w=w)
    y = x.clone()
    y[2], y[5] = float("nan"), float("inf")
    s = t.clone()
    s[2] = float("nan")
    z = y.detach().requires_grad_()
    loss = sft.distill_loss(z, s, i, row_weight=w)
    g, = torch.autograd.grad(loss, z)
    assert torch.equal(loss, want[0]) and torch.equal(g, want[1])
    y[3, 4] = float("nan")
    z = y.detach().requires_grad_()
    rows = sft.distill_loss(z, s, i, row_weight=w, reduction="none")
    g, = torch.autograd.grad(rows, z, torch.ones_like(rows))
    assert rows.isnan().nonzero().flatten().tolist() == [3] and bool(g[3].isnan().all()) and not bool(g[[0, 1, 2, 4, 5]].isnan().any())


@pytest.mark.parametrize("dtype", TYPES)
def test_logits_of_minus_infinity(gpu, dtype):
    """A masked part of the vocabulary has no share; a teacher's entry there makes the loss infinite, one of share 0 not."""
    x, (t, i) = randn(4, 200, dtype=dtype), entries(4, 200, 3, absent=False)
    i[:] = torch.tensor([150, 160, 170], device="cuda")
    x[:, :100] = -math.inf
    check(x, t, i)
    i[1, 2] = 5
    z = x.detach().requires_grad_()
    rows = sft.distill_loss(z, t, i, reduction="none")
    g, = torch.autograd.grad(rows.sum(), z)
    assert rows.isinf().nonzero().flatten().tolist() == [1] and bool(g.isfinite().all())
    t[1, 2] = -1e4
    assert bool(sft.distill_loss(z, t, i, reduction="none").isfinite().all())
    x[2] = torch.finfo(dtype).min
    check(x, t, i)
    x[3] = -math.inf
    assert sft.distill_loss(x, t, i, reduction="none").isnan().tolist() == [False, False, False, True]


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows_count(gpu, dtype):
    x, (t, i) = randn(5, 40, dtype=dtype), entries(5, 40, 3)
    for w, j in ((torch.zeros(5, device="cuda"), i), (None, torch.full_like(i, -1))):
        for reduction in ("mean", "sum", "none"):
            z = x.detach().requires_grad_()
            loss = sft.distill_loss(z, t, j, row_weight=w, reduction=reduction)
            g, = torch.autograd.grad(loss.sum(), z)
            assert not bool(loss.any()) and not bool(g.any())
    for shape in ((0,), (2, 0)):
        z = torch.zeros(*shape, 40, dtype=dtype, device="cuda", requires_grad=True)
        for reduction in ("mean", "sum", "none"):
            loss = sft.distill_loss(z, torch.zeros(*shape, 3, device="cuda"), torch.zeros(*shape, 3, device="cuda").long(), reduction=reduction)
            g, = torch.autograd.grad(loss.sum(), z)
            assert float(loss.detach().sum()) == 0 and g.shape == z.shape
    assert float(sft.distill_loss(x, t[:, :0], i[:, :0])) == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_upstream_gradients(gpu, dtype):
    """Any factor gives the factor's gradient with one rounding, a graph kept for a second pass too."""
    x, (t, i) = randn(30, 700, dtype=dtype), entries(30, 700, 5)
    for g in (1.0, 0.5, 1024.0, -7.0, 0.0):
        check(x, t, i, g=torch.tensor(g, device="cuda"))
    z = x.detach().requires_grad_()
    loss = sft.distill_loss(z, t, i)
    first, = torch.autograd.grad(loss, z, retain_graph=True)
    keep = first.clone()
    first.zero_()
    second, = torch.autograd.grad(loss, z, retain_graph=True)
    third, = torch.autograd.grad(loss, z, torch.tensor(2.0, device="cuda"))
    # (a subnormal is off by half a step, twice that when doubled)
    step = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert torch.equal(second, keep) and float((third.double() - 2 * keep.double()).abs().max()) <= 1.5 * step
    z.grad = None
    (sft.distill_loss(z, t, i) * 0.5 + sft.distill_loss(z, t, i) * 0.5).backward()
    assert float((z.grad.double() - keep.double()).abs().max()) <= float(keep.double().abs().max()) * torch.finfo(dtype).eps


def test_against_differences(gpu):
    x, (t, i) = randn(3, 50), entries(3, 50, 4, absent=False)
    z = x.detach().requires_grad_()
    g, = torch.autograd.grad(sft.distill_loss(z, t, i, temperature=2.0, reduction="sum"), z)
    x = x.double()
    for r in range(3):
        for j in range(0, 50, 7):
            h, at = 1e-4, float(x[r, j])
            x[r, j] = at + h
            up = rows64(x, t, i, 2.0)[0].sum()
            x[r, j] = at - h
            down = rows64(x, t, i, 2.0)[0].sum()
            x[r, j] = at
            # (a third difference over 6 is below h^2 here, and float32's own part)
            assert abs(float((up - down) / (2 * h)) - float(g[r, j])) < 1e-5


def test_the_same_bits_each_time_and_streams(gpu):
    x, (t, i) = randn(400, 5003, dtype=torch.bfloat16), entries(400, 5003, 32)

    def one():
        z = x.detach().requires_grad_()
        loss = sft.distill_loss(z, t, i)
        return loss.detach(), *torch.autograd.grad(loss, z)
    first = one()
    torch.cuda.synchronize()
    got = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            got.append(one())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for other in got for a, b in zip(first, other))


@pytest.mark.parametrize("dtype", TYPES)
def test_captured(gpu, dtype):
    """In one graph, and as two graphs of which the second is replayed with other factors and a gradient changed by hand."""
    x, (t, i) = randn(20, 900, dtype=dtype).requires_grad_(), entries(20, 900, 6)
    g = torch.ones((), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(sft.distill_loss(x, t, i), x, g)
    torch.cuda.current_stream().wait_stream(side)

    def want(factor):
        z = x.detach().clone().requires_grad_()
        return torch.autograd.grad(sft.distill_loss(z, t, i), z, torch.tensor(factor, device="cuda"))[0]

    one = torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        loss = sft.distill_loss(x, t, i)
        grad, = torch.autograd.grad(loss, x, g)
    ahead, behind = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ahead):
        later = sft.distill_loss(x, t, i)
    with torch.cuda.graph(behind, pool=ahead.pool()):
        split, = torch.autograd.grad(later, x, g)
    for seed, factor in ((5, 1.0), (6, 3.0), (7, 1.0)):
        with torch.no_grad():
            x.copy_(randn(20, 900, seed=seed, dtype=dtype))
        g.fill_(factor)
        one.replay()
        assert torch.equal(grad, want(factor))
        ahead.replay()
        behind.replay()
        assert torch.equal(split, want(factor)) and torch.equal(later, loss)
        split.zero_()
        g.fill_(1.0)
        behind.replay()
        assert torch.equal(split, want(1.0))


def test_kept_tensors_on_the_host(gpu):
    x, (t, i) = torch.zeros(5, 9, 210, dtype=torch.bfloat16, device="cuda")[:, :-1, :200].copy_(randn(5, 8, 200)), entries(40, 200, 4)
    t, i = t.view(5, 8, 4), i.view(5, 8, 4)
    want = check(x, t, i)[1]
    with torch.autograd.graph.save_on_cpu():
        assert torch.equal(check(x, t, i)[1], want)
        check(x, t, i, g=torch.tensor(3.0, device="cuda"))


def test_a_wait_that_runs_out_is_reported(gpu):
    """Parts of a row that never come: the rows are NaN, it is counted, and the next call is as if nothing had been."""
    from superfloat.python_b200 import _lib
    x, (t, i) = randn(5, 9000), entries(5, 9000, 3, absent=False)
    want = sft.distill_loss(x, t, i, reduction="none")
    before = sft.tensor_failures()
    _lib.load().sfb_wide_wait_limit(2000, 1)
    try:
        z = x.detach().requires_grad_()
        loss = sft.distill_loss(z, t, i)
        g, = torch.autograd.grad(loss, z)
    finally:
        _lib.load().sfb_wide_wait_limit(0, 0)
    assert bool(loss.isnan()) and bool(g.isnan().all()) and sft.tensor_failures() > before
    assert torch.equal(sft.distill_loss(x, t, i, reduction="none"), want)


def test_refusals(gpu):
    x, t, i = randn(4, 30), randn(4, 3), torch.zeros(4, 3, dtype=torch.int64, device="cuda")
    for bad in (dict(reduction="max"), dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=-1.0)):
        with pytest.raises(ValueError):
            sft.distill_loss(x, t, i, **bad)
    for args in ((x.double(), t, i), (x, t.double(), i), (x, t, i.short()), (x, t.requires_grad_(), i)):
        with pytest.raises(SFTypeError):
            sft.distill_loss(*args)
    t = t.detach()
    for args in ((x, t[:3], i), (x, t[:, :2], i), (x, t, i.cpu()), (x, t.cpu(), i), (x[..., :0], t, i),
                 (x, torch.zeros(4, 1025, device="cuda"), torch.zeros(4, 1025, device="cuda").long())):
        with pytest.raises(SFShapeError):
            sft.distill_loss(*args)
    with pytest.raises(SFShapeError):
        sft.distill_loss(x, t, i, row_weight=torch.ones(5, device="cuda"))
    with pytest.raises(SFTypeError):
        sft.distill_loss(x, t, i, row_weight=torch.ones(4, device="cuda").double())
    loss = sft.distill_loss(x.requires_grad_(), t, i)
    g, = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    import torch.autograd.forward_ad as fa
    with fa.dual_level(), pytest.raises(SFUnsupportedError):
        sft.distill_loss(fa.make_dual(x.detach(), x.detach()), t, i)
