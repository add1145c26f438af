"""Converted layers on the tensor cores as a program uses them: conversion,
training with the straight-through gradient and AdamW (float32 and sf8 states),
graph capture, the compile backend, packing and serving."""
import copy

import pytest
import torch
import torch.nn as nn

import superfloat.python_b200.torch as sft
from superfloat.python_b200._errors import SFTypeError, SFUnsupportedError

pytestmark = pytest.mark.gpu


class Block(nn.Module):
    """An embedding, a residual two-layer network and a head, as a language model's."""

    def __init__(self, vocab=96, d=64, h=160):
        super().__init__()
        self.emb = nn.Embedding(vocab, d)
        self.up, self.down, self.head = nn.Linear(d, h), nn.Linear(h, d), nn.Linear(d, vocab, bias=False)

    def forward(self, ids):
        x = self.emb(ids)
        x = x + self.down(torch.nn.functional.gelu(self.up(x)))
        return self.head(x)


def model(dtype=torch.bfloat16, bits="sf8", scale="per_channel"):
    torch.manual_seed(0)
    return sft.convert(Block().cuda().to(dtype), dtype=bits, accumulate="tensor", scale=scale)


def batch(seed=0, n=4, t=50):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, 96, (n, t), generator=g, device="cuda")


def loss_of(net, ids):
    logits = net(ids[:, :-1])
    return nn.functional.cross_entropy(logits.flatten(0, 1).float(), ids[:, 1:].flatten())


class Rounded(torch.autograd.Function):
    """The sf8 weight of the rule in 64 bits, straight through."""

    @staticmethod
    def forward(ctx, w):
        s = (w.abs().amax(1) / (127 / 128)).float().double()
        return torch.round(w / s[:, None] * 128).clamp(-127, 127) / 128 * s[:, None]

    @staticmethod
    def backward(ctx, g):
        return g


def test_training_gradients_against_the_formula(gpu):
    """Every parameter's gradient against the same network in 64 bits.  Each layer rounds its result, dz and dx to
    bf16, 2^-9 of a tensor's norm at most each; three layers forward and back have nine of them, the embedding, the
    sum and the loss's gradient three more, and the gelu's slope and the residual's two paths no more than double a
    relative error: 12 x 2 x 2^-9 < 5 %."""
    net = model()
    ids = batch()
    loss_of(net, ids).backward()
    ref = {n: p.detach().double().requires_grad_() for n, p in net.named_parameters()}
    f = nn.functional
    q = Rounded.apply
    x = f.embedding(ids[:, :-1], ref["emb.weight"])
    h = f.gelu(f.linear(x, q(ref["up.weight"]), ref["up.bias"]))
    x = x + f.linear(h, q(ref["down.weight"]), ref["down.bias"])
    f.cross_entropy(f.linear(x, q(ref["head.weight"])).flatten(0, 1), ids[:, 1:].flatten()).backward()
    for n, p in net.named_parameters():
        rel = float((p.grad.double() - ref[n].grad).norm() / ref[n].grad.norm())
        assert rel < 0.05, (n, rel)


@pytest.mark.parametrize("state", ["float32", "sf8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_training_run(gpu, dtype, state):
    """Forward, loss, backward and step together: everything stays finite and every parameter moves."""
    net = model(dtype, "sf6", "per_tensor")
    before = copy.deepcopy(net.state_dict())
    opt = sft.AdamW(net.parameters(), lr=1e-3, state=state)
    for i in range(8):
        opt.zero_grad()
        loss = loss_of(net, batch(i))
        loss.backward()
        opt.step()
        assert bool(loss.detach().isfinite())
    for n, p in net.named_parameters():
        assert bool(p.isfinite().all()) and not torch.equal(p, before[n]), n
        m, v = opt.moments(p)
        assert m.shape == p.shape and bool((v >= 0).all())
    kinds = {st["exp_avg"].dtype for st in opt.state.values()}
    assert kinds == ({torch.int8, torch.float32} if state == "sf8" else {torch.float32})


def test_a_captured_training_step(gpu):
    """Forward, backward and a capturable step in one graph, replayed on new batches: the eager run's parameters."""
    nets = [model(), model()]
    opts = [sft.AdamW(n.parameters(), lr=1e-3, state="sf8", capturable=True) for n in nets]
    static = batch(0)

    def step(net, opt, ids):
        opt.zero_grad(set_to_none=False)
        loss_of(net, ids).backward()
        opt.step()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                     # the first step off the default stream, as captures want it
        step(nets[0], opts[0], static)
    torch.cuda.current_stream().wait_stream(side)
    step(nets[1], opts[1], batch(0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(nets[0], opts[0], static)
    for i in range(1, 4):
        static.copy_(batch(i))
        graph.replay()
        step(nets[1], opts[1], batch(i))
    torch.cuda.synchronize()
    for p, r in zip(nets[0].parameters(), nets[1].parameters()):
        assert torch.equal(p, r)


def test_hugging_face_conv1d(gpu):
    """A Conv1D's (in, out) weight, converted and trained: the linear's results and gradients, transposed."""
    class Conv1D(nn.Module):
        def __init__(self, nf, nx):
            super().__init__()
            self.nf, self.nx = nf, nx
            self.weight = nn.Parameter(torch.randn(nx, nf, device="cuda").bfloat16() * 0.1)
            self.bias = nn.Parameter(torch.randn(nf, device="cuda").bfloat16())

    torch.manual_seed(1)
    conv = Conv1D(48, 80)
    lin = nn.Linear(80, 48).cuda().bfloat16()
    with torch.no_grad():
        lin.weight.copy_(conv.weight.t())
        lin.bias.copy_(conv.bias)
    a, b = (sft.convert(m, dtype="sf8", accumulate="tensor") for m in (nn.Sequential(conv), nn.Sequential(lin)))
    x = torch.randn(70, 80, device="cuda").bfloat16()
    ya, yb = a(x), b(x)
    assert torch.equal(ya, yb)
    g = torch.randn_like(ya)
    ya.backward(g)
    yb.backward(g)
    assert torch.equal(a[0].weight.grad, b[0].weight.grad.t()) and torch.equal(a[0].bias.grad, b[0].bias.grad)
    pa, pb = sft.pack(a), sft.pack(b)
    assert torch.equal(pa(x), pb(x)) and torch.equal(pa[0].codes, pb[0].codes)


def test_packing(gpu):
    """A packed model gives the layers' own results, at one byte a weight; its state_dict loads into another."""
    net = model()
    ids = batch(3)
    with torch.no_grad():
        want = net(ids)
        packed = sft.pack(net)
        assert torch.equal(packed(ids), want)         # 200 rows: the same product
        few = packed(ids[:1, :3])                     # 3 rows: straight from the codes
        assert float((few - want[:1, :3]).abs().max()) <= 2 ** -7 * float(want.abs().max())
    assert type(packed.up).__name__ == "SFPackedLinear" and packed.up.codes.dtype == torch.int8
    assert type(net.up).__name__ == "SFLinear"
    other = sft.pack(model())
    other.load_state_dict(packed.state_dict())
    with torch.no_grad():
        assert torch.equal(other(ids), want)
    half = copy.deepcopy(packed).half()               # the scales stay float32
    assert half.up.scale.dtype == torch.float32 and half.up.codes.dtype == torch.int8
    with torch.no_grad():
        assert half(ids).dtype == torch.float16
    moved = copy.deepcopy(packed).cpu().cuda()
    with torch.no_grad():
        assert torch.equal(moved(ids), want)
    x = torch.randn(5, 64, device="cuda").bfloat16()
    r = torch.randn(5, 160, device="cuda").bfloat16()
    fused = packed.up(x, activation="silu", residual=r)
    assert fused.shape == (5, 160) and fused.dtype == torch.bfloat16


def test_shared_layers_are_packed_once(gpu):
    lin = nn.Linear(16, 16).cuda().bfloat16()
    net = sft.convert(nn.Sequential(lin, nn.ReLU(), lin), dtype="sf8", accumulate="tensor")
    packed = sft.pack(net)
    assert packed[0] is packed[2]


def test_the_compile_backend_runs_the_eager_layers(gpu):
    net = model()
    ids = batch(4)
    with torch.no_grad():
        want = net(ids)
        got = torch.compile(net, backend="superfloat")(ids)
    assert torch.equal(got, want)
    rep = sft.compile_report()
    assert sorted(op for _, op, _, _ in rep.on_device) == ["linear_tensor"] * 3


def test_the_custom_op_and_its_gradient(gpu):
    x = torch.randn(90, 64, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(40, 64, device="cuda") * 0.1).requires_grad_()
    b = torch.randn(40, device="cuda").requires_grad_()
    g = torch.randn(90, 40, device="cuda").bfloat16()
    for bias in (b, None):
        wanted = [t for t in (x, w, bias) if t is not None]
        y = torch.ops.sf.linear_tensor(x, w, bias, 8, "per_channel", "layer")
        z = sft.tensor_linear(x, w, bias)
        assert torch.equal(y, z)
        for p, q in zip(torch.autograd.grad(y, wanted, g), torch.autograd.grad(z, wanted, g)):
            assert torch.equal(p, q)


def test_functional_and_layer_refusals(gpu):
    lin = nn.Linear(16, 8).cuda()
    x = torch.randn(4, 16, device="cuda")
    with pytest.raises(SFTypeError, match="float32"):     # a float32 model: the message names the other modes
        sft.convert(lin, dtype="sf8", accumulate="tensor")(x)
    y = sft.linear(x.bfloat16(), lin.weight, lin.bias, dtype="sf8", scale="per_channel", accumulate="tensor")
    assert y.dtype == torch.bfloat16 and torch.equal(y, sft.tensor_linear(x.bfloat16(), lin.weight, lin.bias))
    with pytest.raises(SFUnsupportedError):
        sft.linear(x.bfloat16(), lin.weight, dtype="sf16", accumulate="tensor")


def test_no_status_is_recorded(gpu):
    net = model()
    with sft.capture_status() as st, torch.no_grad():
        net(batch(5))
    assert st == {}
