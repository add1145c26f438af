"""The gated product on the B200 against its formula in 64 bits.

Tolerances, with u = 2^-24, e = finfo(type).eps and the float32 sums' error of test_gpu_tensor_linear (S the sum of the
products' magnitudes, (K / 16 + 16) 2^-23 S, three roundings for scale and bias): g and z are off by `off`; the
activation by 1.13 off + 2e-6 (1 + |g|), its slope by 1.2 off + 4e-6; h by the two products of an error and the other
factor, u |h|, and half a step of its type.  dg = dh u act'(g) and du = dh act(g) by the same and 3 u of themselves, and
as operands by half a step of the type; the products sum these errors' magnitudes.
"""
import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200._errors import SFShapeError, SFTypeError, SFUnsupportedError
from test_gpu_tensor_linear import act64, close, codes64, randn, sum_error

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
ACTS = ["silu", "gelu", "gelu_tanh", "relu", None]
U = 2.0 ** -24
# rows, channels, features: one of each, groups of 16 channels that end early, few rows, tiles of both widths
SIZES = [(1, 1, 1), (1, 16, 16), (2, 3, 5), (7, 40, 24), (16, 130, 64), (17, 64, 129), (33, 96, 256), (48, 257, 72), (49, 40, 128),
         (128, 128, 64), (129, 259, 65), (200, 515, 1000), (515, 300, 96), (1000, 17, 2049), (300, 1031, 520)]


def product64(x, codes, s, bits, bias):
    wq = codes * (s * 2.0 ** (1 - bits))[:, None]
    x = x.detach().double()
    z = x @ wq.T
    b = torch.zeros_like(s) if bias is None else bias.detach().double()
    return z + b, sum_error(x.shape[1], x.abs() @ wq.abs().T) + 3 * U * (z.abs() + b.abs()), wq


def forward64(x, cg, sg, cu, su, bits, bg, bu, act):
    """(h, its tolerance without the last rounding), and what the backward pass needs."""
    g, off_g, wg = product64(x, cg, sg, bits, bg)
    u, off_u, wu = product64(x, cu, su, bits, bu)
    a = act64(g, act)
    tol_a = 1.13 * off_g + (0 if act in (None, "relu") else 2e-6) * (1 + g.abs())
    h = a * u
    tol = u.abs() * tol_a + a.abs() * off_u + tol_a * off_u + U * h.abs()
    return h, tol, (g, off_g, u, off_u, a, tol_a, wg, wu)


def backward64(x, kept, act, dh, dtype, top):
    """[(gradient, tolerance without the last rounding)] of x, both weights and both biases."""
    g, off_g, u, off_u, a, tol_a, wg, wu = kept
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    zz = g.clone().requires_grad_()
    s, = torch.autograd.grad(act64(zz, act).sum(), zz)
    off_s = torch.zeros_like(g) if act in (None, "relu") else 1.2 * off_g + 4e-6
    dh = dh.double()
    dg, du = dh * u * s, dh * a
    e_g = dh.abs() * (u.abs() * off_s + s.abs() * off_u + off_s * off_u) + 3 * U * dg.abs()
    e_u = dh.abs() * tol_a + U * du.abs()
    x = x.detach().double()
    M, N = dg.shape
    out, dx, tol = [], 0, 0
    for d, e, w in ((dg, e_g, wg), (du, e_u, wu)):
        dx = dx + d @ w
        # d s / top: the subnormal step is one of top
        tol = tol + (e + half * (d.abs() + e)) @ w.abs() * (1 + 2.0 ** -20) + tiny * top * (w.abs() > 0).double().sum(0)
        tol = tol + sum_error(2 * N, d.abs() @ w.abs())
        out.append((d.T @ x, (e + half * (d.abs() + e) + tiny).T @ x.abs() + sum_error(M, d.abs().T @ x.abs())))
    out += [(d.sum(0), e.sum(0) + (M + 2) * U * d.abs().sum(0)) for d, e in ((dg, e_g), (du, e_u))]
    return [(dx, tol), *out]


def weights(n, k, dtype=torch.float32, seed=2):
    return randn(n, k, seed=seed, std=k ** -0.5, dtype=dtype), randn(n, k, seed=seed + 20, std=k ** -0.5, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_packed(gpu, m, n, k, dtype):
    x = randn(m, k, seed=1, dtype=dtype)
    for i, act in enumerate(ACTS):
        bits = [8, 4, 6, 8, 7][i]
        gate, up = (sft.pack_weight(w, f"sf{bits}") for w in weights(n, k))
        bg = randn(n, seed=3, std=0.3, dtype=[torch.float32, dtype][i % 2]) if i != 1 else None
        bu = randn(n, seed=4, std=0.3, dtype=[dtype, torch.float32][i % 2]) if i < 3 else None
        h = sft.tensor_gated(x, gate, up, bg, bu, activation=act)
        want, tol, _ = forward64(x, gate.codes.double(), gate.scale.double(), up.codes.double(), up.scale.double(), bits, bg, bu, act)
        assert h.shape == (m, n) and h.dtype == dtype
        close(h, want, tol, dtype)


@pytest.mark.parametrize("wscale", ["per_channel", "per_tensor"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_training(gpu, m, n, k, dtype, wscale):
    for i, act in enumerate(ACTS):
        bits = [8, 4, 6, 8, 7][i]
        w_dtype = [dtype, torch.float32][i % 2]
        x = randn(m, k, seed=1, dtype=dtype).requires_grad_()
        gate, up = (w.requires_grad_() for w in weights(n, k, w_dtype))
        bg = randn(n, seed=3, std=0.3, dtype=[torch.float32, dtype][i % 2]).requires_grad_() if i != 1 else None
        bu = randn(n, seed=4, std=0.3, dtype=[dtype, torch.float32][i % 2]).requires_grad_() if i < 3 else None
        dh = randn(m, n, seed=5, dtype=dtype)
        (cg, sg), (cu, su) = codes64(gate, bits, wscale), codes64(up, bits, wscale)
        want, tol, kept = forward64(x, cg, sg, cu, su, bits, bg, bu, act)
        if act == "relu":
            dh = dh * (kept[0].abs() > 1e-2)
        h = sft.tensor_gated(x, gate, up, bg, bu, activation=act, dtype=f"sf{bits}", scale=wscale)
        close(h.detach(), want, tol, dtype)
        h.backward(dh)
        pairs = backward64(x, kept, act, dh, dtype, max(float(sg.max()), float(su.max())))
        for t, pair in zip((x, gate, up, bg, bu), pairs):
            if t is not None:
                assert t.grad.dtype == t.dtype and t.grad.shape == t.shape
                close(t.grad, *pair, t.dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_products(gpu, dtype):
    """Sizes at which tiles are shared by pairs of SMs in all products, ragged in each direction."""
    m, n, k = 2100, 2107, 2201
    x = randn(m, k, seed=1, dtype=dtype).requires_grad_()
    gate, up = (w.requires_grad_() for w in weights(n, k, dtype))
    bg, bu = randn(n, seed=3, std=0.3).requires_grad_(), randn(n, seed=4, std=0.3).requires_grad_()
    dh = randn(m, n, seed=5, dtype=dtype)
    (cg, sg), (cu, su) = codes64(gate, 8, "per_channel"), codes64(up, 8, "per_channel")
    want, tol, kept = forward64(x, cg, sg, cu, su, 8, bg, bu, "silu")
    h = sft.tensor_gated(x, gate, up, bg, bu)
    close(h.detach(), want, tol, dtype)
    h.backward(dh)
    for t, pair in zip((x, gate, up, bg, bu), backward64(x, kept, "silu", dh, dtype, max(float(sg.max()), float(su.max())))):
        close(t.grad, *pair, t.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 100])
def test_layouts(gpu, rows, dtype):
    """Rows of a wider buffer, odd offsets, transposed inputs, strided codes, scales and biases: the same bits."""
    x = randn(rows, 3, 100, dtype=dtype)
    gate, up = (sft.pack_weight(w) for w in weights(50, 100))
    bg, bu = randn(50, seed=3, dtype=dtype), randn(50, seed=4)
    want = sft.tensor_gated(x, gate, up, bg, bu)
    assert want.shape == (rows, 3, 50)
    for off in (0, 1, 8):
        xs = torch.zeros(rows, 3, 117, dtype=dtype, device="cuda")[..., off:off + 100].copy_(x)
        assert torch.equal(sft.tensor_gated(xs, gate, up, bg, bu), want)
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    codes = torch.zeros(50, 117, dtype=torch.int8, device="cuda")[:, 5:105].copy_(up.codes)
    us = sft.SFPackedWeight(codes, torch.zeros(100, device="cuda")[::2].copy_(up.scale), 8)
    bs = torch.zeros(101, dtype=dtype, device="cuda")[1::2].copy_(bg)
    for args in ((xt, gate, up, bg, bu), (x, gate, us, bg, bu), (x, gate, up, bs, bu)):
        assert torch.equal(sft.tensor_gated(*args), want)
    assert sft.tensor_gated(x[1, 2], gate, up, bg, bu).shape == (50,)
    wide = torch.cat([w for w in weights(50, 100)])         # both weights as halves of one
    full = sft.tensor_gated(x, *weights(50, 100), bg, bu)
    assert torch.equal(sft.tensor_gated(x, wide[:50], wide[50:], bg, bu), full) and torch.equal(full, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_each_gradient_alone(gpu, dtype):
    """Only what is asked for, within the tolerances of all together; a shared gradient of ones."""
    m, n, k = 70, 40, 96
    args = [randn(m, k, dtype=dtype), *weights(n, k), randn(n, seed=3), randn(n, seed=4)]
    dh = randn(m, n, seed=5, dtype=dtype)
    (cg, sg), (cu, su) = codes64(args[1], 8, "per_channel"), codes64(args[2], 8, "per_channel")
    _, _, kept = forward64(args[0], cg, sg, cu, su, 8, *args[3:], "silu")
    pairs = backward64(args[0], kept, "silu", dh, dtype, max(float(sg.max()), float(su.max())))
    for wanted in ([0], [1], [2], [3], [4], [1, 2], [1, 3], [0, 4], [2, 3, 4], [0, 1, 2, 3, 4]):
        t = [a.detach().clone().requires_grad_(i in wanted) for i, a in enumerate(args)]
        got = torch.autograd.grad(sft.tensor_gated(*t), [t[i] for i in wanted], dh)
        for i, g in zip(wanted, got):
            close(g, *pairs[i], t[i].dtype)
    t = [a.detach().clone().requires_grad_() for a in args]
    ones = torch.autograd.grad(sft.tensor_gated(*t), t, torch.ones_like(dh))
    for a, b in zip(torch.autograd.grad(sft.tensor_gated(*t).sum(), t), ones):
        assert torch.equal(a, b)
    same = args[1].detach().clone().requires_grad_()           # one weight in both places
    x = args[0].detach()
    got, = torch.autograd.grad(sft.tensor_gated(x, same, same), same, dh)
    _, _, kept = forward64(x, cg, sg, cg, sg, 8, None, None, "silu")
    (_, _), (a, ta), (b, tb), *_ = backward64(x, kept, "silu", dh, dtype, float(sg.max()))
    close(got, a + b, (ta + tb) + 3 * U * (a.abs() + b.abs()), torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_weights_pass_gradients_to_the_rest(gpu, dtype):
    for m, n, k in ((9, 24, 40), (130, 33, 65)):
        x = randn(m, k, dtype=dtype).requires_grad_()
        gate, up = (sft.pack_weight(w) for w in weights(n, k))
        b = randn(n, seed=3).requires_grad_()
        dh = randn(m, n, seed=5, dtype=dtype)
        sft.tensor_gated(x, gate, up, None, b).backward(dh)
        args = [t.double() for p in (gate, up) for t in (p.codes, p.scale)]
        _, _, kept = forward64(x, *args, 8, None, b, "silu")
        pairs = backward64(x, kept, "silu", dh, dtype, max(float(gate.scale.max()), float(up.scale.max())))
        close(x.grad, *pairs[0], dtype)
        close(b.grad, *pairs[4], torch.float32)


@pytest.mark.parametrize("rows", [3, 200])
def test_empty_and_not_finite(gpu, rows):
    gate, up = (w.bfloat16().requires_grad_() for w in weights(20, 16))
    x = torch.zeros(2, 0, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    b = randn(20).requires_grad_()
    h = sft.tensor_gated(x, gate, up, b)
    h.sum().backward()
    assert h.shape == (2, 0, 20) and x.grad.shape == x.shape and not any(bool(t.grad.any()) for t in (gate, up, b))
    gate, up = (sft.pack_weight(w) for w in weights(48, 64))
    x = randn(rows, 64, dtype=torch.bfloat16)
    clean = sft.tensor_gated(x, gate, up)
    x[rows // 2, 5] = float("nan")
    h = sft.tensor_gated(x, gate, up)
    hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
    hit[rows // 2] = True
    assert bool(h[hit].isnan().all()) and torch.equal(h[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_and_small_scales(gpu, dtype):
    """A weight of 1e-5 beside rows of zeros (whose scale is 1), large inputs: gradients keep their range."""
    m, n, k = 40, 33, 64
    gate, up = weights(n, k)
    gate, up = gate * 1e-3, up * 1e-5
    gate[3], up[7], up[3] = 0, 0, 0
    x = (randn(m, k, seed=1) * 100).to(dtype).requires_grad_()
    gate.requires_grad_(), up.requires_grad_()
    dh = (randn(m, n, seed=5) * 100).to(dtype)
    (cg, sg), (cu, su) = codes64(gate, 8, "per_channel"), codes64(up, 8, "per_channel")
    want, tol, kept = forward64(x, cg, sg, cu, su, 8, None, None, "silu")
    h = sft.tensor_gated(x, gate, up)
    close(h.detach(), want, tol, dtype)
    h.backward(dh)
    top = max(float(s[c.abs().amax(1) > 0].max()) for c, s in ((cg, sg), (cu, su)))
    for t, pair in zip((x, gate, up), backward64(x, kept, "silu", dh, dtype, top)):
        close(t.grad, *pair, t.dtype)


def test_a_large_second_product(gpu):
    """Products past float16's range are kept as they are."""
    x = torch.full((3, 16), 3e4, device="cuda").bfloat16().requires_grad_()
    w = sft.pack_weight(torch.eye(16, device="cuda") * 127 / 128)
    up = sft.pack_weight(torch.eye(16, device="cuda") * 127 * 8)
    h = sft.tensor_gated(x, w, up, activation="relu")
    g, = torch.autograd.grad(h, x, torch.ones_like(h))
    # dh act'(g) u Wg + dh act(g) Wu = 2 g u / x: 6e7 x 1016, of which bf16's roundings take less than 2 %
    assert bool(g.isfinite().all()) and float(g.min()) > 2 * 0.98 * 3e4 * 127 * 8 * 127 / 128


def test_captured_and_two_streams(gpu):
    x = randn(200, 128, dtype=torch.bfloat16).requires_grad_()
    gate, up = (w.requires_grad_() for w in weights(96, 128))
    dh = randn(200, 96, seed=5, dtype=torch.bfloat16)

    def one():
        h = sft.tensor_gated(x, gate, up)
        return h.detach(), *torch.autograd.grad(h, (x, gate, up), dh)
    want = one()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(one())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for other in got for a, b in zip(want, other))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = one()
    for seed in (7, 8):
        with torch.no_grad():
            x.copy_(randn(200, 128, seed=seed, dtype=torch.bfloat16))
            gate.copy_(weights(96, 128, seed=seed)[0])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, one()))


def test_kept_tensors_on_the_host(gpu):
    x, dh = randn(70, 65, dtype=torch.float16), randn(70, 24, seed=5, dtype=torch.float16)
    gate, up = weights(24, 65)
    for xs in (x, torch.zeros(70, 80, dtype=torch.float16, device="cuda")[:, :65].copy_(x)):
        t = [xs.detach().requires_grad_(), gate.clone().requires_grad_(), up.clone().requires_grad_()]
        want = torch.autograd.grad(sft.tensor_gated(*t), t, dh)
        with torch.autograd.graph.save_on_cpu():
            got = torch.autograd.grad(sft.tensor_gated(*t), t, dh)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals(gpu):
    x, (gate, up) = randn(4, 32, dtype=torch.bfloat16), weights(16, 32)
    p, q = sft.pack_weight(gate), sft.pack_weight(up, "sf6")
    for args in ((x, p, up), (x, p, q), (x, gate, up.bfloat16()), (x.float(), gate, up), (x, gate.double(), up.double())):
        with pytest.raises(SFTypeError):
            sft.tensor_gated(*args)
    for args in ((x, gate, up[:15]), (x[:, :31], gate, up), (x, gate, up.cpu()), (x.cpu(), gate, up), (x, gate[0], up[0]),
                 (x, gate, up, torch.zeros(15, device="cuda")), (x, gate, up, None, torch.zeros(17, device="cuda")),
                 (x, gate, up, None, torch.zeros(16))):
        with pytest.raises(SFShapeError):
            sft.tensor_gated(*args)
    with pytest.raises(ValueError):
        sft.tensor_gated(x, gate, up, activation="tanh")
    with pytest.raises(ValueError):
        sft.tensor_gated(x, gate, up, scale="per_row")
    with pytest.raises(SFUnsupportedError):
        sft.tensor_gated(x, gate, up, dtype="sf16")
    h = sft.tensor_gated(x.requires_grad_(), gate, up)
    g, = torch.autograd.grad(h, x, torch.ones_like(h), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    import torch.autograd.forward_ad as fa
    with fa.dual_level(), pytest.raises(SFUnsupportedError):
        sft.tensor_gated(fa.make_dual(x.detach(), x.detach()), gate, up)
