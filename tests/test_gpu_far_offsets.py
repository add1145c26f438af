"""Sizes whose elements pass 2^31: the last rows against their formulas, gradients that sum over all rows against their
parts.  Tolerances as in the operators' own tests, where these are derived."""
import pytest
import torch

import superfloat.python_b200.torch as sft
import test_gpu_distill as distill
import test_gpu_gated as gated
import test_gpu_norm as norm
from test_gpu_tensor_linear import close, codes64, randn

pytestmark = pytest.mark.gpu
TAIL = 5


def big(m, n, dtype=torch.bfloat16, seed=0):
    """Rows that repeat, but for the last ones."""
    part = randn(4096, n, seed=seed, dtype=dtype)
    out = part.repeat((m + 4095) // 4096, 1)[:m]
    out[-TAIL:] = randn(TAIL, n, seed=seed + 1, dtype=dtype)
    return out


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def test_norm(gpu):
    m, d = 530_000, 4096
    x, dy = big(m, d), big(m, d, seed=5)
    assert x.numel() > 2 ** 31
    w, b = 1 + randn(d, seed=3, std=0.3), randn(d, seed=4)
    y, gx, gw, gb = norm.run(x, w, b, dy)
    want = norm.formula(x[-TAIL:], w, b, dy[-TAIL:])
    norm.close(y[-TAIL:], *want[0])
    norm.close(gx[-TAIL:], *want[1])
    # dw and db: of the repeated rows so often, and of the last ones; n roundings of a sum as norm.formula has them
    x, dy = x.detach(), dy.detach()
    whole, rest = divmod(m - TAIL, 4096)
    (_, _, (w0, t0), (b0, u0)) = norm.formula(x[:4096], w, b, dy[:4096])
    (_, _, (w1, t1), (b1, u1)) = norm.formula(x[:rest], w, b, dy[:rest])
    (_, _, (w2, t2), (b2, u2)) = want
    n = (m / 18 + 100) / (4096 / 18 + 100)
    norm.close(gw, whole * w0 + w1 + w2, n * whole * t0 + n * whole * t1 + n * whole * t2)
    norm.close(gb, whole * b0 + b1 + b2, n * whole * u0 + n * whole * u1 + n * whole * u2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_distill(gpu, dtype):
    m, v, k = 43_000, 50_257, 6
    logits = big(m, v, dtype)
    assert logits.numel() > 2 ** 31
    t, i = distill.entries(m, v, k, seed=2, absent=False)
    i[-2, 1:] = -1
    z = logits.requires_grad_()
    loss = sft.distill_loss(z, t, i, reduction="sum")
    g, = torch.autograd.grad(loss, z, torch.tensor(64.0, device="cuda"))
    row, tol, grad, gtol, _ = distill.rows64(z[-TAIL:], t[-TAIL:], i[-TAIL:], 1.0)
    distill.close(g[-TAIL:], 64 * grad, 64 * (gtol + 20 * distill.U * grad.abs()))
    with torch.no_grad():
        rows = sft.distill_loss(logits, t, i, reduction="none")
    distill.close(rows[-TAIL:], row, tol + 4 * distill.U * row.abs())
    # the sum of the rows' losses, 256 running sums of m / 256 and their own
    assert abs(float(loss.detach()) - float(rows.double().sum())) <= (m / 256 + 20) * distill.U * float(rows.double().abs().sum())


def test_gated(gpu):
    m, n, k = 66_000, 16_400, 64
    x, dh = big(m, k), big(m, n, seed=5)
    gate, up = (w.requires_grad_() for w in gated.weights(n, k, torch.bfloat16))
    x.requires_grad_()
    h = sft.tensor_gated(x, gate, up)
    gx, = torch.autograd.grad(h, x, dh)
    assert m * 2 * n > 2 ** 31
    (cg, sg), (cu, su) = codes64(gate, 8, "per_channel"), codes64(up, 8, "per_channel")
    want, tol, kept = gated.forward64(x[-TAIL:], cg, sg, cu, su, 8, None, None, "silu")
    close(h[-TAIL:].detach(), want, tol, torch.bfloat16)
    (pair, *_) = gated.backward64(x[-TAIL:], kept, "silu", dh[-TAIL:], torch.bfloat16, max(float(sg.max()), float(su.max())))
    close(gx[-TAIL:], *pair, torch.bfloat16)
    # the weights' gradients take the same rows: those of the last ones alone differ by the others', which are masked out
    with torch.no_grad():
        dh[:-TAIL] = 0
    gg, gu = torch.autograd.grad(sft.tensor_gated(x, gate, up), (gate, up), dh)
    _, pg, pu, *_ = gated.backward64(x[-TAIL:], kept, "silu", dh[-TAIL:], torch.bfloat16, max(float(sg.max()), float(su.max())))
    close(gg, *pg, torch.bfloat16)
    close(gu, *pu, torch.bfloat16)
