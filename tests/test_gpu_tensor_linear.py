"""The tensor-core linear on the B200 against its formula in 64 bits.

Tolerances, per element, with e = finfo(type).eps (a rounding is off by at most
e / 2 of the value) and S the sum of the products' magnitudes:

* the float32 sum: 16 products a step, so at most K / 16 + 16 additions, each
  off by at most one unit (the tensor cores truncate) of a partial sum below S:
  (K / 16 + 16) 2^-23 S;
* the scale and the bias: three float32 roundings, 3 x 2^-24 (|z| + |b|);
* the activation: slope at most 1.13, and its approximation below 2e-6 (1 + |z|)
  (erf's 1.5e-7 absolute, and approximate exponentials and quotients);
* the result's rounding: e / 2 |y|.

Backward: dz is rounded to the type, e / 2 |dz|, before either product; act'
reads z in fp16, off by 2^-11 |z|, and |z act''(z)| is below 0.7 for all four,
so act' is off by at most 0.7 x 2^-11 + 1.2 x the error of z + 4e-6 (relu's step
is kept out: no |z| below 1e-2 gets a gradient there).  Both errors go through
the products as sums of magnitudes.
"""
import math

import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200 import _lib
from superfloat.python_b200._errors import SFShapeError, SFTypeError, SFUnsupportedError

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]
SIZES = [(1, 1, 1), (1, 16, 16), (2, 3, 5), (7, 40, 24), (16, 130, 64), (17, 64, 129), (33, 96, 256), (48, 257, 72), (49, 40, 128), (128, 256, 64),
         (129, 259, 65), (200, 515, 1000), (515, 300, 96), (1000, 33, 2049)]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * std).to(dtype)


def act64(z, act):
    f = torch.nn.functional
    return {None: lambda v: v.clone(), "relu": f.relu, "gelu": f.gelu, "silu": f.silu,
            "gelu_tanh": lambda v: f.gelu(v, approximate="tanh")}[act](z)


def codes64(w, bits, wscale):
    """(codes, scales) of a float weight from the rule, in 64 bits; the scale is kept as float32."""
    w = w.detach().double()
    one = 2.0 ** (bits - 1)
    top = w.abs().amax(1) if wscale == "per_channel" else w.abs().amax().expand(w.shape[0])
    s = torch.where(top > 0, top / ((one - 1) / one), torch.ones_like(top)).float().double()
    return torch.round(w / s[:, None] * one).clamp(1 - one, one - 1), s


def sum_error(K, mags):
    return (K / 16 + 16) * 2.0 ** -23 * mags


def forward64(x, codes, s, bits, bias, act, residual):
    """(y, tolerance without the last rounding, z, error of z)."""
    wq = codes * (s * 2.0 ** (1 - bits))[:, None]
    x = x.detach().double()
    z = x @ wq.T
    b = torch.zeros_like(s) if bias is None else bias.detach().double()
    off = sum_error(x.shape[1], x.abs() @ wq.abs().T) + 3 * 2.0 ** -24 * (z.abs() + b.abs())
    z = z + b
    y = act64(z, act)
    tol = 1.13 * off + (0 if act in (None, "relu") else 2e-6) * (1 + z.abs())
    if residual is not None:
        y = y + residual.detach().double()
        tol = tol + 2.0 ** -24 * (y.abs() + residual.detach().double().abs())
    return y, tol, z, off


def close(got, want, tol, dtype):
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps          # a step of the subnormals
    bound = tol * (1 + half) + half * want.abs() + tiny
    ratio = ((got.double() - want).abs() / bound).max() if got.numel() else torch.zeros(())
    assert float(ratio) <= 1, float(ratio)


# --- codes ------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("wscale", ["per_channel", "per_tensor"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [4, 6, 8])
def test_pack_weight(gpu, bits, dtype, wscale):
    w = randn(37, 301, dtype=dtype)
    w[3] = 0
    w[5] *= 1e-3
    p = sft.pack_weight(w, f"sf{bits}", wscale)
    codes, s = codes64(w, bits, wscale)
    assert torch.equal(p.scale.double(), s) and torch.equal(p.codes.double(), codes)
    err = (p.dequantize().double() - w.double()).abs() / (s[:, None] * 2.0 ** (1 - bits))
    assert float(err.max()) <= 0.5 + 1e-5
    assert p.bits == bits and p.shape == w.shape


def test_pack_weight_ties_go_to_even(gpu):
    """Weights on the borders of two codes: amax 127 makes the scale 128 and the quotient exact."""
    w = torch.arange(-127, 127.5, 0.5, device="cuda")[None]
    assert torch.equal(sft.pack_weight(w).codes[0].double(), torch.round(w[0].double()))
    w3 = (w.double() * 3).float()                     # scale 384: the reciprocal is not exact, the ties are
    assert torch.equal(sft.pack_weight(w3).codes[0].double(), torch.round(w[0].double()))


def test_pack_weight_layouts_and_rows_that_are_not_finite(gpu):
    w = randn(70, 50)
    for view in (w.t(), w[:, 3:40], w[::2]):
        p, q = sft.pack_weight(view), sft.pack_weight(view.contiguous())
        assert torch.equal(p.codes, q.codes) and torch.equal(p.scale, q.scale)
    w[4, 7], w[6, 1] = float("nan"), float("inf")
    p = sft.pack_weight(w)
    x = randn(3, 50, dtype=torch.bfloat16)
    y = sft.tensor_linear(x, p)
    assert y.isnan().any(0).nonzero().flatten().tolist() == [4, 6] and bool(y[:, [4, 6]].isnan().all())


# --- forward ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_packed_forward(gpu, m, n, k, dtype):
    x = randn(m, k, seed=1, dtype=dtype)
    p = sft.pack_weight(randn(n, k, seed=2, std=k ** -0.5))
    for i, act in enumerate(ACTS):
        bias = randn(n, seed=3, dtype=[torch.float32, dtype][i % 2]) if i != 1 else None
        res = randn(m, n, seed=4, dtype=dtype) if i % 2 else None
        y = sft.tensor_linear(x, p, bias, activation=act, residual=res)
        want, tol, _, _ = forward64(x, p.codes.double(), p.scale.double(), 8, bias, act, res)
        assert y.shape == (m, n) and y.dtype == dtype
        close(y, want, tol, dtype)


@pytest.mark.parametrize("bits", [4, 5, 6, 7, 8])
def test_every_code_and_width(gpu, bits):
    """Codes over the whole range, x one-hot and scaled: each product alone, exactly."""
    M = 2 ** (bits - 1) - 1
    codes = torch.arange(-M, M + 1, device="cuda", dtype=torch.int8).view(1, -1).repeat(9, 1)
    scale = 2.0 ** torch.arange(-4, 5, device="cuda").float()
    K = codes.shape[1]
    p = sft.SFPackedWeight(codes, scale, bits)
    for rows in (K, 4):
        x = (torch.eye(K, device="cuda") * 2)[:rows].to(torch.bfloat16)
        y = sft.tensor_linear(x, p)
        want = 2 * codes.double().t()[:rows] * scale.double() * 2.0 ** (1 - bits)
        assert torch.equal(y.double(), want.to(torch.bfloat16).double())


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(gpu, dtype):
    """Leading dimensions, rows of a wider buffer, odd offsets, transposed inputs, strided codes: the same bits."""
    x = randn(4, 30, 100, dtype=dtype)
    w = sft.pack_weight(randn(50, 100, std=0.1))
    b = randn(50, dtype=dtype, seed=3)
    r = randn(4, 30, 50, dtype=dtype, seed=4)
    want = sft.tensor_linear(x, w, b, activation="silu", residual=r)
    assert want.shape == (4, 30, 50)
    wide = torch.zeros(4, 30, 109, dtype=dtype, device="cuda")
    for off in (0, 1, 8):
        xs = wide[..., off:off + 100]
        xs.copy_(x)
        assert torch.equal(sft.tensor_linear(xs, w, b, activation="silu", residual=r), want)
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    rt = r.transpose(0, 2).contiguous().transpose(0, 2)
    rw = torch.zeros(4, 30, 57, dtype=dtype, device="cuda")[..., 3:53].copy_(r)
    bw = torch.zeros(101, dtype=dtype, device="cuda")[1::2].copy_(b)
    codes = torch.zeros(50, 117, dtype=torch.int8, device="cuda")[:, 5:105].copy_(w.codes)
    ws = sft.SFPackedWeight(codes, torch.zeros(100, device="cuda")[::2].copy_(w.scale), 8)
    wt = sft.SFPackedWeight(w.codes.t().contiguous().t(), w.scale, 8)
    for args in ((xt, w, b, r), (x, w, b, rt), (x, w, b, rw), (x, w, bw, r), (x, ws, b, r), (x, wt, b, r)):
        assert torch.equal(sft.tensor_linear(*args[:3], activation="silu", residual=args[3]), want)
    one = sft.tensor_linear(x[1, 2], w, b, activation="silu", residual=r[1, 2])
    assert one.shape == (50,)
    close(one, *forward64(x[1, 2][None], w.codes.double(), w.scale.double(), 8, b, "silu", r[1, 2][None])[:2], dtype)
    broadcast = x[:1, :1].expand(3, 5, 100)
    y = sft.tensor_linear(broadcast, w)
    assert torch.equal(y, y[:1, :1].expand(3, 5, 50))


def test_empty_batches(gpu):
    w = randn(20, 16, dtype=torch.bfloat16).requires_grad_()
    x = torch.zeros(2, 0, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    b = randn(20).requires_grad_()
    y = sft.tensor_linear(x, w, b, activation="gelu")
    assert y.shape == (2, 0, 20)
    y.sum().backward()
    assert x.grad.shape == x.shape and float(w.grad.abs().sum()) == 0 and float(b.grad.abs().sum()) == 0


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_not_finite_inputs_stay_in_their_rows(gpu, rows):
    x = randn(rows, 64, dtype=torch.bfloat16)
    w = sft.pack_weight(randn(48, 64, std=0.1))
    clean = sft.tensor_linear(x, w, activation="gelu")
    x[rows // 2, 5] = float("nan")
    y = sft.tensor_linear(x, w, activation="gelu")
    hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
    hit[rows // 2] = True
    nz = w.codes[:, 5] != 0                            # a code of 0 times NaN is NaN too
    assert bool(y[hit].isnan().all()) and bool(nz.any()) and torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", TYPES)
def test_far_pre_activations(gpu, dtype):
    """Large |z|: activations at their asymptotes, without a NaN; gradients there too."""
    w = sft.pack_weight(torch.eye(8, device="cuda") * 127 / 128)
    z = torch.tensor([-3e4, -300.0, -30.0, -6.0, 6.0, 30.0, 300.0, 3e4], device="cuda").to(dtype)
    x = torch.diag(z).requires_grad_()
    for act in ACTS:
        y = sft.tensor_linear(x, w, activation=act)
        g, = torch.autograd.grad(y, x, torch.ones_like(y))
        want, tol, zz, _ = forward64(x, w.codes.double(), w.scale.double(), 8, None, act, None)
        close(y.detach(), want, tol, dtype)
        assert bool(g.isfinite().all())
        d = torch.diag(g).double() / (127 / 128)
        far = torch.tensor([0.0, 0.0, 0.0], device="cuda", dtype=torch.float64)
        if act is not None:
            assert torch.allclose(d[:3], far, atol=1e-4) and torch.allclose(d[5:], far + 1, atol=2e-2)


# --- backward ---------------------------------------------------------------------------------------------------


def backward64(x, codes, s, bits, bias, act, dy, dtype, w_dtype, b_dtype):
    """Gradients of x, the weight and the bias with their tolerances (last rounding apart)."""
    half = torch.finfo(dtype).eps / 2
    _, _, z, off = forward64(x, codes, s, bits, bias, act, None)
    zz = z.clone().requires_grad_()
    d, = torch.autograd.grad(act64(zz, act).sum(), zz)
    dy = dy.double()
    dz = dy * d
    off_d = torch.zeros_like(d) if act is None else (0 if act == "relu" else 1) * (0.7 * 2.0 ** -11 + 1.2 * off + 4e-6)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    e_dz = dy.abs() * off_d
    e_op = e_dz + half * (dz.abs() + e_dz) + tiny        # as an operand
    wq = codes * (s * 2.0 ** (1 - bits))[:, None]
    x = x.detach().double()
    M, N = dz.shape
    # dz s / max s: the subnormal step is one of max s
    e_opx = (e_dz + half * (dz.abs() + e_dz)) @ wq.abs() + tiny * (s.max() * codes.abs() * 2.0 ** (1 - bits)).sum(0)
    gx = (dz @ wq, e_opx * (1 + 2.0 ** -20) + sum_error(N, dz.abs() @ wq.abs()))
    gw = (dz.T @ x, e_op.T @ x.abs() + sum_error(M, dz.abs().T @ x.abs()))
    gb = (dz.sum(0), e_dz.sum(0) + (M + 2) * 2.0 ** -24 * dz.abs().sum(0))
    return gx, gw, gb


def close_grad(got, pair, dtype):
    close(got, pair[0], pair[1], dtype if dtype != torch.float32 else torch.float32)


@pytest.mark.parametrize("wscale", ["per_channel", "per_tensor"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_training(gpu, m, n, k, dtype, wscale):
    for i, act in enumerate(ACTS):
        bits = [8, 4, 8, 6, 7][i]
        w_dtype = [dtype, torch.float32][i % 2]
        x = randn(m, k, seed=1, dtype=dtype).requires_grad_()
        w = randn(n, k, seed=2, std=k ** -0.5, dtype=w_dtype).requires_grad_()
        b = randn(n, seed=3, std=0.3, dtype=[torch.float32, dtype][i % 2]).requires_grad_() if i != 2 else None
        r = randn(m, n, seed=4, dtype=dtype).requires_grad_() if i > 2 else None
        dy = randn(m, n, seed=5, dtype=dtype)
        codes, s = codes64(w, bits, wscale)
        want, tol, z, _ = forward64(x, codes, s, bits, b, act, r)
        if act == "relu":
            dy = dy * (z.abs() > 1e-2)
        y = sft.tensor_linear(x, w, b, activation=act, residual=r, dtype=f"sf{bits}", scale=wscale)
        close(y.detach(), want, tol, dtype)
        y.backward(dy)
        gx, gw, gb = backward64(x, codes, s, bits, b, act, dy, dtype, w.dtype, None)
        close_grad(x.grad, gx, dtype)
        assert w.grad.dtype == w_dtype
        close_grad(w.grad, gw, w_dtype)
        if b is not None:
            assert b.grad.dtype == b.dtype
            close_grad(b.grad, gb, b.dtype)
        if r is not None:
            assert torch.equal(r.grad, dy)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_products(gpu, dtype):
    """Sizes at which tiles are shared by pairs of SMs in all three products, ragged in each direction."""
    m, n, k = 4100, 4107, 4201
    x = randn(m, k, seed=1, dtype=dtype).requires_grad_()
    w = randn(n, k, seed=2, std=k ** -0.5, dtype=dtype).requires_grad_()
    b = randn(n, seed=3, std=0.3).requires_grad_()
    r, dy = randn(m, n, seed=4, dtype=dtype), randn(m, n, seed=5, dtype=dtype)
    codes, s = codes64(w, 8, "per_channel")
    want, tol, _, _ = forward64(x, codes, s, 8, b, "gelu", r)
    y = sft.tensor_linear(x, w, b, activation="gelu", residual=r)
    close(y.detach(), want, tol, dtype)
    y.backward(dy)
    gx, gw, gb = backward64(x, codes, s, 8, b, "gelu", dy, dtype, w.dtype, None)
    close_grad(x.grad, gx, dtype)
    close_grad(w.grad, gw, dtype)
    close_grad(b.grad, gb, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_weight_passes_gradients_to_the_rest(gpu, dtype):
    x = randn(33, 40, dtype=dtype).requires_grad_()
    p = sft.pack_weight(randn(24, 40, seed=2, std=0.2))
    b = randn(24, seed=3).requires_grad_()
    r = randn(33, 24, seed=4, dtype=dtype).requires_grad_()
    dy = randn(33, 24, seed=5, dtype=dtype)
    sft.tensor_linear(x, p, b, activation="gelu", residual=r).backward(dy)
    gx, _, gb = backward64(x, p.codes.double(), p.scale.double(), 8, b, "gelu", dy, dtype, None, None)
    close_grad(x.grad, gx, dtype)
    close_grad(b.grad, gb, torch.float32)
    assert torch.equal(r.grad, dy)


def test_each_gradient_alone(gpu):
    """Only the gradients asked for, each the bits it has beside the others; shared and strided output gradients."""
    args = [randn(50, 64, dtype=torch.bfloat16), randn(30, 64, seed=1, std=0.1), randn(30, seed=2)]
    dy = randn(50, 30, seed=3, dtype=torch.bfloat16)
    for act in (None, "silu"):
        for wscale in ("per_channel", "per_tensor"):
            full = [a.clone().requires_grad_() for a in args]
            y = sft.tensor_linear(*full, activation=act, scale=wscale)
            want = torch.autograd.grad(y, full, dy, retain_graph=True)
            again = torch.autograd.grad(y, full, dy.t().contiguous().t())
            assert all(torch.equal(a, b) for a, b in zip(want, again))
            for i in range(3):
                part = [a.clone().requires_grad_(j == i) for j, a in enumerate(args)]
                y = sft.tensor_linear(*part, activation=act, scale=wscale)
                got, = torch.autograd.grad(y, [part[i]], dy)
                assert torch.equal(got, want[i])
            part = [a.clone().requires_grad_() for a in args]
            y = sft.tensor_linear(*part, activation=act, scale=wscale)
            got = torch.autograd.grad(y.sum(), part)          # an expanded gradient of ones
            ones = torch.autograd.grad(sft.tensor_linear(*part, activation=act, scale=wscale), part,
                                       torch.ones_like(dy))
            assert all(torch.equal(a, b) for a, b in zip(got, ones))


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_gradient_against_differences(gpu, act):
    """The directional derivative of sum(y c) in x and the bias from the kernel's gradients, against central
    differences of the formula in 64 bits.  A gradient's element is within e / 2 of its value and of dz's sums
    (the bounds above); 4 e over the sum of magnitudes covers both."""
    dtype = torch.bfloat16
    x, w = randn(32, 48, dtype=dtype), sft.pack_weight(randn(40, 48, seed=1, std=0.2))
    b, c = randn(40, seed=2), randn(32, 40, seed=3, dtype=dtype)
    dx, db = randn(32, 48, seed=4).double(), randn(40, seed=5).double()
    wq = w.codes.double() * (w.scale.double() / 128)[:, None]

    def f(h):
        return (act64((x.double() + h * dx) @ wq.T + b.double() + h * db, act) * c.double()).sum()

    h = 1e-4
    slope = float((f(h) - f(-h)) / (2 * h))
    xr, br = x.clone().requires_grad_(), b.clone().requires_grad_()
    sft.tensor_linear(xr, w, br, activation=act).backward(c)
    got = float((xr.grad.double() * dx).sum() + (br.grad.double() * db).sum())
    mags = float((c.double().abs() @ wq.abs() * dx.abs()).sum() * 1.13 + (c.double().abs().sum(0) * 1.13 * db.abs()).sum())
    assert abs(got - slope) <= 4 * torch.finfo(dtype).eps * mags


def test_small_scales_do_not_leave_fp16(gpu):
    """A weight of 1e-5: dz s is below fp16's normal range, dx is not lost."""
    x = randn(20, 32, dtype=torch.float16).requires_grad_()
    w = randn(24, 32, seed=1, std=1e-5)
    dy = randn(20, 24, seed=2, dtype=torch.float16)
    for wscale in ("per_channel", "per_tensor"):
        p = w.clone().requires_grad_()
        x.grad = None
        sft.tensor_linear(x, p, scale=wscale).backward(dy * 100)
        codes, s = codes64(w, 8, wscale)
        gx, gw, _ = backward64(x, codes, s, 8, None, None, dy * 100, torch.float16, None, None)
        close_grad(x.grad, gx, torch.float16)
        close_grad(p.grad, gw, torch.float32)


# --- how it is called -------------------------------------------------------------------------------------------


def test_refusals(gpu):
    x = randn(4, 32, dtype=torch.bfloat16)
    w = randn(16, 32, dtype=torch.bfloat16)
    p = sft.pack_weight(w)
    for bits in ("sf9", "sf16"):
        with pytest.raises(SFUnsupportedError, match="sf4..sf8"):
            sft.tensor_linear(x, w, dtype=bits)
        with pytest.raises(SFUnsupportedError):
            sft.pack_weight(w, bits)
    with pytest.raises(SFTypeError, match="float32"):
        sft.tensor_linear(x.float(), w)
    with pytest.raises(SFTypeError, match="float64"):
        sft.tensor_linear(x, w.double())
    with pytest.raises(SFTypeError, match="residual"):
        sft.tensor_linear(x, w, residual=torch.zeros(4, 16, device="cuda"))
    with pytest.raises(SFTypeError, match="bias"):
        sft.tensor_linear(x, w, torch.zeros(16, dtype=torch.int32, device="cuda"))
    for bad in (dict(bias=torch.zeros(15, device="cuda")), dict(residual=x[:, :16][:3]), dict(residual=x[:1, :16]),
                dict(bias=torch.zeros(16))):
        with pytest.raises(SFShapeError):
            sft.tensor_linear(x, w, **bad)
    with pytest.raises(SFShapeError, match="features"):
        sft.tensor_linear(x[:, :31], w)
    with pytest.raises(SFShapeError):
        sft.tensor_linear(x.cpu(), w)
    with pytest.raises(SFShapeError):
        sft.tensor_linear(x, w.cpu())
    with pytest.raises(SFShapeError):
        sft.tensor_linear(x, w[0])
    with pytest.raises(ValueError, match="activation"):
        sft.tensor_linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="scale"):
        sft.tensor_linear(x, w, scale="per_row")
    with pytest.raises(SFShapeError):
        sft.SFPackedWeight(p.codes, p.scale[:3])
    with pytest.raises(SFTypeError):
        sft.SFPackedWeight(p.codes.float(), p.scale)
    with pytest.raises(SFUnsupportedError):
        sft.SFPackedWeight(p.codes, p.scale, 9)
    with pytest.raises(SFShapeError):
        sft.pack_weight(w[:0])


@pytest.mark.parametrize("rows", [1, 24, 200])
def test_another_stream_and_a_graph(gpu, rows):
    x = randn(rows, 128, dtype=torch.bfloat16)
    w = randn(96, 128, seed=1, dtype=torch.bfloat16, std=0.1)
    p = sft.pack_weight(w)
    want = [sft.tensor_linear(x, q, activation="silu") for q in (w, p)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [sft.tensor_linear(x, q, activation="silu") for q in (w, p)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = torch.zeros_like(x)
    graphs, outs = [], []
    for q in (w, p):                                   # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sft.tensor_linear(static, q, activation="silu"))
        graphs.append(g)
    static.copy_(x)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_a_captured_training_step(gpu):
    """Forward and backward captured together, replayed on new inputs: the eager step's bits."""
    x = randn(40, 64, dtype=torch.bfloat16)
    w = randn(48, 64, seed=1, std=0.1).requires_grad_()
    b = randn(48, seed=2).requires_grad_()
    dy = randn(40, 48, seed=3, dtype=torch.bfloat16)
    static = torch.zeros_like(x)

    def step(inp):
        y = sft.tensor_linear(inp, w, b, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, [w, b], dy))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(static)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(static)
    static.copy_(x)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(out, step(x)))


def test_what_the_backward_pass_kept(gpu):
    """x changed in place before the backward pass is an error; the weight may change (its codes are kept); a second
    derivative is refused."""
    x = randn(20, 64, dtype=torch.bfloat16)
    w = randn(24, 64, seed=1, std=0.1).requires_grad_()
    y = sft.tensor_linear(x, w)
    want, = torch.autograd.grad(y, w, torch.ones_like(y), retain_graph=True)
    with torch.no_grad():
        w.mul_(2)
    again, = torch.autograd.grad(y, w, torch.ones_like(y), retain_graph=True)
    assert torch.equal(want, again)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, w, torch.ones_like(y))
    xr = randn(20, 64, dtype=torch.bfloat16).requires_grad_()
    y = sft.tensor_linear(xr, w, activation="gelu")
    g, = torch.autograd.grad(y.float().square().sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|twice|differentiate"):
        g.float().sum().backward()


def test_calls_on_two_streams_at_once(gpu):
    """Training passes of two layers interleaved on two streams: each the bits it has alone."""
    def layer(seed):
        x = randn(900, 512, seed=seed, dtype=torch.bfloat16).requires_grad_()
        w = randn(700, 512, seed=seed + 1, std=0.05).requires_grad_()
        dy = randn(900, 700, seed=seed + 2, dtype=torch.bfloat16)
        return x, w, dy

    def run(x, w, dy):
        y = sft.tensor_linear(x, w, activation="silu")
        return (y.detach(), *torch.autograd.grad(y, [x, w], dy))

    sets = [layer(0), layer(10)]
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(*sets[i]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for r in g:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


def test_runs_repeat(gpu):
    x = randn(700, 512, dtype=torch.bfloat16).requires_grad_()
    w = randn(600, 512, seed=1, std=0.05).requires_grad_()
    b = randn(600, seed=2).requires_grad_()
    dy = randn(700, 600, seed=3, dtype=torch.bfloat16)

    def step():
        y = sft.tensor_linear(x, w, b, activation="gelu_tanh")
        return (y.detach(), *torch.autograd.grad(y, [x, w, b], dy))

    first = step()
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, step()))


@pytest.mark.parametrize("m,n", [(300, 200), (4100, 4100)])        # one SM to a tile, and pairs
def test_a_wait_that_runs_out_leaves_nan(gpu, m, n):
    """With every wait of the products bounded by 1000 polls and the first made on a barrier that nothing arrives
    on, the call returns, its outputs are NaN, the CTAs are counted, and the next call is whole."""
    x = randn(m, 256, dtype=torch.bfloat16)
    w = sft.pack_weight(randn(n, 256, seed=1, std=0.1))
    want = sft.tensor_linear(x, w)
    before = sft.tensor_failures()
    try:
        _lib.load().sfb_wide_wait_limit(1000, 1)
        y = sft.tensor_linear(x, w)
    finally:
        _lib.load().sfb_wide_wait_limit(0, 0)
    assert bool(y.isnan().all()) and sft.tensor_failures() > before
    assert torch.equal(sft.tensor_linear(x, w), want)


def test_large_offsets(gpu):
    """Rows whose offsets pass 2^31 elements, in x, the residual and the result."""
    M, K, N = 2_200_000, 8, 1000
    w = sft.pack_weight(randn(N, K, seed=1))
    x = randn(M, K, dtype=torch.bfloat16)
    res = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    res[-1] = 5
    y = sft.tensor_linear(x, w, residual=res)
    for rows in (slice(0, 300), slice(M - 300, M)):
        want, tol, _, _ = forward64(x[rows], w.codes.double(), w.scale.double(), 8, None, None, res[rows])
        close(y[rows], want, tol, torch.bfloat16)
    assert math.prod(y.shape) > 2 ** 31


@pytest.mark.parametrize("rows,channels", [(1, 40), (65, 31), (700, 130), (2100, 64)])
def test_the_bias_gradient_is_the_same_alone_and_beside_the_products(rows, channels):
    """Its partial sums are added up by a kernel of their own where the weight's gradient is not wanted, else beside
    that product: the same sums in the same order."""
    x, w, b = randn(rows, 48, seed=1), randn(channels, 48, seed=2), randn(channels, seed=3)
    dy, grads = randn(rows, channels, seed=4).bfloat16(), []
    for want_x, want_w in ((False, False), (True, False), (False, True), (True, True)):
        xs, ws, bs = (t.bfloat16().requires_grad_(want) for t, want in ((x, want_x), (w, want_w), (b, True)))
        sft.tensor_linear(xs, ws, bs, activation="relu").backward(dy)
        grads.append(bs.grad)
    assert all(torch.equal(g, grads[0]) for g in grads[1:])
    open_ = sft.tensor_linear(x.bfloat16(), w.bfloat16(), b.bfloat16(), activation="relu") > 0
    exact = (dy.double() * open_).sum(0)
    # float32 sums of `rows` terms, then one rounding to bf16
    bound = dy.double().abs().sum(0) * rows * 2.0 ** -24 + exact.abs() * 2.0 ** -8
    assert ((grads[0].double() - exact).abs() <= bound).all()
