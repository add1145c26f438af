"""Norms, gated blocks and the distillation loss as a program uses them together: a converted student tuned against its
float teacher, captured, compiled, packed and served."""
import copy

import pytest
import torch
import torch.nn as nn

import superfloat.python_b200.torch as sft
from test_gpu_tensor_training import Rounded

pytestmark = pytest.mark.gpu


class Gated(nn.Module):
    def __init__(self, d, h):
        super().__init__()
        self.gate_proj, self.up_proj = nn.Linear(d, h), nn.Linear(d, h, bias=False)
        self.down_proj, self.act_fn = nn.Linear(h, d), nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Student(nn.Module):
    """An embedding, a norm, a gated residual block, a norm and a head of an odd vocabulary."""

    def __init__(self, vocab=97, d=72, h=120):
        super().__init__()
        self.emb, self.norm, self.mlp = nn.Embedding(vocab, d), nn.LayerNorm(d), Gated(d, h)
        self.last, self.head = nn.LayerNorm(d), nn.Linear(d, vocab, bias=False)

    def forward(self, ids):
        x = self.emb(ids)
        return self.head(self.last(x + self.mlp(self.norm(x))))


def models(dtype=torch.bfloat16, seed=0):
    """(teacher, student converted from it)"""
    torch.manual_seed(seed)
    net = Student().cuda().to(dtype)
    with torch.no_grad():
        for n in (net.norm, net.last):
            n.weight.uniform_(0.5, 1.5)
            n.bias.uniform_(-0.5, 0.5)
    return net, sft.convert(net, dtype="sf8", accumulate="tensor", scale="per_channel", fuse=True)


def batch(seed=0, n=3, t=41):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, 97, (n, t), generator=g, device="cuda")
    mask = torch.rand(n, t, generator=g, device="cuda") < 0.8
    mask[0] = False                                    # a sequence of nothing but padding
    return ids, mask


@torch.no_grad()
def taught(teacher, ids, k=8):
    top = teacher(ids).float().topk(k)
    return top.values + 2 * torch.randn(top.values.shape, generator=torch.Generator("cuda").manual_seed(9), device="cuda"), top.indices


def loss_of(net, ids, mask, top):
    return sft.distill_loss(net(ids), *top, temperature=2.0, row_weight=mask)


def formula(net, ids, mask, top):
    """The loss and every parameter's gradient, in 64 bits."""
    p = {n: t.detach().double().requires_grad_() for n, t in net.named_parameters()}
    f, q = nn.functional, Rounded.apply
    x = f.embedding(ids, p["emb.weight"])
    d = x.shape[-1:]
    a = f.layer_norm(x, d, p["norm.weight"], p["norm.bias"])
    h = f.silu(f.linear(a, q(p["mlp.gate_proj.weight"]), p["mlp.gate_proj.bias"])) * f.linear(a, q(p["mlp.up_proj.weight"]))
    x = x + f.linear(h, q(p["mlp.down_proj.weight"]), p["mlp.down_proj.bias"])
    z = f.linear(f.layer_norm(x, d, p["last.weight"], p["last.bias"]), q(p["head.weight"])) / 2
    t = torch.log_softmax(top[0].double() / 2, -1)
    rows = 4 * (t.exp() * (t - torch.log_softmax(z, -1).gather(-1, top[1]))).sum(-1)
    loss = (rows * mask).sum() / mask.sum()
    return loss, dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


@pytest.mark.parametrize("dtype,part", [(torch.bfloat16, 1), (torch.float16, 8)])
def test_gradients_against_the_formula(gpu, dtype, part):
    """Each operator rounds its result and its gradients to the type, half a step (2^-9 or 2^-12) of a tensor's norm at
    most each: on the longest path six results, one more for the residual, and nine gradients and operands.  The gate,
    the norms' scales and the softmax multiply a relative error by no more than 2.5: 16 x 2.5 x 2^-9 < 8 %."""
    teacher, net = models(dtype)
    ids, mask = batch()
    top = taught(teacher, ids)
    loss = loss_of(net, ids, mask, top)
    scale = 1024.0 if dtype == torch.float16 else 1.0
    (loss * scale).backward()
    want, grads = formula(net, ids, mask, top)
    want = float(want.detach())
    assert abs(float(loss.detach()) - want) < 0.08 / part * want
    for n, p in net.named_parameters():
        rel = float((p.grad.double() / scale - grads[n]).norm() / grads[n].norm())
        assert rel < 0.08 / part, (n, rel)


@pytest.mark.parametrize("state", ["float32", "sf8"])
def test_a_captured_step_is_the_eager_one(gpu, state):
    """Forward, loss, backward and AdamW in one graph, replayed on new batches."""
    teacher, net = models()
    net.emb.weight.requires_grad_(False)               # (its gradient is torch's, added up by atomics)
    nets = [net, copy.deepcopy(net)]
    opts = [sft.AdamW([p for p in n.parameters() if p.requires_grad], lr=1e-3, state=state, capturable=True) for n in nets]
    ids, mask = batch()
    values, places = taught(teacher, ids)

    def step(net, opt, ids, mask, top):
        opt.zero_grad(set_to_none=False)
        loss_of(net, ids, mask, top).backward()
        opt.step()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(nets[0], opts[0], ids, mask, (values, places))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(nets[0], opts[0], ids, mask, (values, places))
    step(nets[1], opts[1], *batch(), taught(teacher, ids))
    for seed in (1, 2):
        new, m = batch(seed)
        top = taught(teacher, new)
        for held, t in ((ids, new), (mask, m), (values, top[0]), (places, top[1])):
            held.copy_(t)
        graph.replay()
        step(nets[1], opts[1], new, m, top)
        for (n, p), q in zip(nets[0].named_parameters(), nets[1].parameters()):
            assert torch.equal(p, q), n


def test_packed_and_served(gpu):
    """One row, few rows and a prompt of the packed model: the eager model's results within bf16's roundings."""
    _, net = models()
    served = sft.pack(net)
    assert isinstance(served.mlp, sft.SFPackedGatedFeedForward) and isinstance(served.mlp.gate_proj, sft.SFPackedLinear)
    assert isinstance(served.norm, sft.SFLayerNorm) and not [n for n in served.state_dict() if n.endswith("gate_proj.weight")]
    with torch.no_grad():
        for n, t in ((1, 1), (3, 5), (4, 60)):
            ids, _ = batch(n, n, t)
            want, got = net(ids).double(), served(ids).double()
            # six results are rounded on either side, and the softmax's logits are one of them: 12 x 2.5 x 2^-9
            assert float((got - want).norm() / want.norm()) < 0.06
    half = copy.deepcopy(served).half()
    assert half.mlp.up_proj.scale.dtype == torch.float32 and bool(half(batch()[0]).isfinite().all())


def test_compiled(gpu):
    """The operators run between a compiled model's graphs: the eager results and gradients."""
    teacher, net = models()
    ids, mask = batch()
    top = taught(teacher, ids)
    loss_of(net, ids, mask, top).backward()
    want = {n: p.grad.clone() for n, p in net.named_parameters()}
    net.zero_grad()
    compiled = torch.compile(net, backend="aot_eager")
    loss_of(compiled, ids, mask, top).backward()
    for n, p in net.named_parameters():
        assert n == "emb.weight" or torch.equal(p.grad, want[n]), n
    with torch.no_grad():
        fast = torch.compile(sft.pack(net), backend="superfloat")
        assert torch.equal(fast(ids), sft.pack(net)(ids))


def test_gradients_are_added_up(gpu):
    """Two halves of a batch, their losses weighted: the whole batch's gradients within the type's roundings."""
    teacher, net = models()
    ids, _ = batch(n=4)
    mask = torch.ones_like(ids, dtype=torch.bool)
    top = taught(teacher, ids)
    loss_of(net, ids, mask, top).backward()
    want = {n: p.grad.clone() for n, p in net.named_parameters()}
    net.zero_grad()
    for part in (slice(0, 2), slice(2, 4)):
        (loss_of(net, ids[part], mask[part], [t[part] for t in top]) * 0.5).backward()
    for n, p in net.named_parameters():
        # every rounding on the path is made twice, of other numbers: 2 x 8 %
        rel = float((p.grad.double() - want[n].double()).norm() / want[n].double().norm())
        assert rel < 0.16, (n, rel)
