"""The cases on which layer norm, the gated feed-forward product over sf codes and the distillation loss are measured.

``run`` computes an operator either in its plain form (elementary torch operations in 32 bits, 64 where a value stands
next to a border) or, where ``own`` is true, through the package's public calls.  Both get the same state.

norm     y = (x - mean) / sqrt(var + eps) w + b over the last dimension.
gated    h = act(x Wg^T + bg) (x Wu^T + bu), both weights as sf codes with a scale a channel (or one a matrix).
         pass "serve": the codes and scales are at hand (packed weights);
         pass "train": the float weights are quantized in the pass.
distill  l = T^2 sum_i p_i (log p_i - log q_i), p the teacher's softmax over the entries that it gives for a row, q the
         student's over the whole vocabulary, both at temperature T; rows have weights.
A training pass returns the result and the gradients of all its inputs.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # one token of a served model before its projection: bound by the latency of the call
        {"name": "norm one token", "op": "norm", "pass": "apply", "m": 1, "n": 768, "type": "bf16", "params": "bf16",
         "affine": "both", "pad": 0},
        # a layer norm of GPT-2-small trained on 8 x 512 tokens, its parameters kept in float32
        {"name": "norm train", "op": "norm", "pass": "train", "m": 4096, "n": 768, "type": "bf16", "params": "f32",
         "affine": "both", "pad": 0},
        # ragged rows of an odd length out of a wider buffer
        {"name": "norm ragged", "op": "norm", "pass": "train", "m": 1023, "n": 1031, "type": "fp16", "params": "fp16",
         "affine": "both", "pad": 5},
        # a wide model's: bound by memory
        {"name": "norm wide", "op": "norm", "pass": "train", "m": 16384, "n": 4096, "type": "bf16", "params": "bf16",
         "affine": "both", "pad": 0},
        # one token of a served model: bound by the two weights' bytes
        {"name": "gated one token", "op": "gated", "pass": "serve", "m": 1, "k": 4096, "n": 8192, "type": "bf16",
         "bits": 8, "act": "silu", "bias": False, "pad": 0},
        # a ragged prompt through odd sizes, sf6 codes, rows of a wider buffer
        {"name": "gated odd prompt", "op": "gated", "pass": "serve", "m": 331, "k": 1031, "n": 2049, "type": "fp16",
         "bits": 6, "act": "gelu_tanh", "bias": True, "pad": 5},
        # a prompt: bound by the tensor cores
        {"name": "gated prompt", "op": "gated", "pass": "serve", "m": 4096, "k": 4096, "n": 8192, "type": "bf16",
         "bits": 8, "act": "silu", "bias": False, "pad": 0},
        # fine-tuning a block of GPT-2-small's width on 8 x 512 tokens
        {"name": "gated train", "op": "gated", "pass": "train", "m": 4096, "k": 768, "n": 2048, "type": "bf16",
         "bits": 8, "act": "silu", "bias": True, "pad": 0, "scale": "per_channel"},
        # fine-tuning a wide block
        {"name": "gated train wide", "op": "gated", "pass": "train", "m": 8192, "k": 2048, "n": 5632, "type": "fp16",
         "bits": 8, "act": "gelu", "bias": False, "pad": 0, "scale": "per_tensor"},
        # a short sequence's step, its loss scaled as float16 asks for
        {"name": "distill few rows", "op": "distill", "pass": "train", "m": 13, "v": 50257, "k": 16, "type": "fp16",
         "temperature": 1.0, "mask": False, "reduction": "mean", "pad": 0},
        # a training step of GPT-2-small's head (a vocabulary of 50257) on 8 x 512 tokens
        {"name": "distill train", "op": "distill", "pass": "train", "m": 4096, "v": 50257, "k": 64, "type": "bf16",
         "temperature": 2.0, "mask": True, "reduction": "mean", "pad": 0},
        # float32 logits, columns of a padded head
        {"name": "distill f32", "op": "distill", "pass": "train", "m": 2047, "v": 32001, "k": 20, "type": "f32",
         "temperature": 1.0, "mask": True, "reduction": "sum", "pad": 31},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "gated", "gated", "distill"])
    dt = rng.choice(["bf16", "fp16"])
    pad = rng.choice([0, 0, 1, 8])
    if kind == "norm":
        dt = rng.choice(["bf16", "fp16", "f32"])
        n = _log(rng, 8, 16384)
        if rng.random() < 0.5:                        # half of the cases are aligned as layers mostly are
            n = 8 * max(1, n // 8)
        return {"op": "norm", "pass": rng.choice(["apply", "train", "train"]), "m": _log(rng, 1, min(16384, 2 ** 26 // n)),
                "n": n, "type": dt, "params": rng.choice(["f32", dt]), "affine": rng.choice(["both", "both", "weight", "none"]),
                "pad": pad}
    if kind == "gated":
        c = {"op": "gated", "pass": rng.choice(["serve", "serve", "train"]), "m": _log(rng, 1, 4096),
             "k": _log(rng, 16, 4096), "n": _log(rng, 16, 5632), "type": dt, "bits": rng.choice([4, 5, 6, 7, 8, 8, 8]),
             "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]), "bias": rng.random() < 0.4, "pad": pad}
        if rng.random() < 0.5:
            c["k"], c["n"] = 16 * max(1, c["k"] // 16), 16 * max(1, c["n"] // 16)
        if c["pass"] == "train":
            c["scale"] = rng.choice(["per_tensor", "per_channel"])
        return c
    v = _log(rng, 300, 50257)
    step = rng.choice(["eval", "train", "train"])
    return {"op": "distill", "pass": step, "m": _log(rng, 1, 4096), "v": v, "k": _log(rng, 1, 256),
            "type": rng.choice(["bf16", "fp16", "f32"]), "temperature": rng.choice([1.0, 1.0, 2.0, 3.5]),
            "mask": rng.random() < 0.6, "reduction": rng.choice(["mean", "sum"] if step == "train" else ["none", "mean"]),
            "pad": pad}


# --- inputs ---------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    dt, m = TYPES[case["type"]], case["m"]
    s = {"case": case}
    if case["op"] == "norm":
        n, pt = case["n"], TYPES[case["params"]]
        # activations with outlier channels and a mean of their own, as a residual stream has
        x = normal(m, n + case["pad"]) * normal(n + case["pad"], std=0.5).exp() + normal(m, 1, std=0.5)
        s["x"] = x.to(dt)[:, :n]
        s["weight"] = (1 + normal(n, std=0.2)).to(pt) if case["affine"] != "none" else None
        s["bias"] = normal(n, std=0.1, dtype=pt) if case["affine"] == "both" else None
        wanted = ("x", "weight", "bias")
        if case["pass"] == "train":
            s["dy"] = normal(m, n, dtype=dt)
    elif case["op"] == "gated":
        k, n = case["k"], case["n"]
        s["x"] = normal(m, k + case["pad"], dtype=dt)[:, :k]
        for name in ("gate", "up"):
            w = normal(n, k, std=k ** -0.5, dtype=dt)
            if case["pass"] == "serve":
                one = 2.0 ** (case["bits"] - 1)
                scale = (w.float().abs().amax(1) / (1 - 1 / one)).clamp_(min=1e-20)
                codes = torch.round(w.float() / scale[:, None] * one).clamp_(1 - one, one - 1).to(torch.int8)
                s[name] = (codes, scale)
            else:
                s[name] = w
            s[name + "_bias"] = normal(n, std=0.1, dtype=dt) if case["bias"] else None
        wanted = ("x", "gate", "up", "gate_bias", "up_bias")
        if case["pass"] == "train":
            s["dy"] = normal(m, n, dtype=dt)
    else:
        v, k = case["v"], case["k"]
        # the teacher's entries: one out of each of k parts of the vocabulary, its logits in falling order, some rows
        # with fewer of them (index -1) and one in about 50 with none
        low = torch.arange(k, device="cuda") * v // k
        size = (torch.arange(1, k + 1, device="cuda") * v // k - low).clamp(min=1)
        index = (low + (torch.rand(m, k, generator=g, device="cuda") * size).long()).clamp_(max=v - 1)
        order = torch.rand(m, k, generator=g, device="cuda").argsort(1)
        index = index.gather(1, order)
        gaps = torch.rand(m, k, generator=g, device="cuda").log_().neg_()
        teacher = 14 - (gaps / torch.arange(1, k + 1, device="cuda")).cumsum(1) * 3
        logits = normal(m, v + case["pad"], std=2.0)
        logits.scatter_add_(1, index, (teacher * 0.6 + normal(m, k)).clamp_(min=0))
        s["logits"] = logits.to(dt)[:, :v]
        kept = (torch.rand(m, generator=g, device="cuda") * 1.5 * k).ceil_().clamp_(max=k)
        kept = torch.where(torch.rand(m, generator=g, device="cuda") < 0.02, torch.zeros_like(kept), kept)
        s["index"] = torch.where(torch.arange(k, device="cuda") < kept[:, None], index, torch.full_like(index, -1))
        s["teacher"] = teacher.to(torch.bfloat16 if case["type"] == "bf16" else torch.float32)
        # prompts and padding do not train
        s["mask"] = torch.rand(m, generator=g, device="cuda") < 0.8 if case["mask"] else None
        wanted = ("logits",)
        # a float16 step scales its loss
        s["dy"] = torch.tensor(1024.0 if case["type"] == "fp16" else 1.0, device="cuda")
    if case["pass"] == "train":
        s["wanted"] = [s[name].requires_grad_() for name in wanted if s[name] is not None]
    return s


# --- one pass -------------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "gated": _own_gated, "distill": _own_distill}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "gated": _plain_gated, "distill": _plain_distill}[op](state)


def _own_norm(s):
    import superfloat.python_b200.torch as sft
    y = sft.layer_norm(s["x"], s["weight"], s["bias"], EPS)
    return y if s["case"]["pass"] == "apply" else [y, *torch.autograd.grad(y, s["wanted"], s["dy"])]


def _own_gated(s):
    import superfloat.python_b200.torch as sft
    c = s["case"]
    if c["pass"] == "serve":
        gate, up = (sft.SFPackedWeight(*s[name], c["bits"]) for name in ("gate", "up"))
        return sft.tensor_gated(s["x"], gate, up, s["gate_bias"], s["up_bias"], activation=c["act"])
    h = sft.tensor_gated(s["x"], s["gate"], s["up"], s["gate_bias"], s["up_bias"], activation=c["act"],
                         dtype="sf%d" % c["bits"], scale=c["scale"])
    return [h, *torch.autograd.grad(h, s["wanted"], s["dy"])]


def _own_distill(s):
    import superfloat.python_b200.torch as sft
    c = s["case"]
    loss = sft.distill_loss(s["logits"], s["teacher"], s["index"], temperature=c["temperature"], row_weight=s["mask"],
                            reduction=c["reduction"])
    return loss if c["pass"] == "eval" else [loss, *torch.autograd.grad(loss, s["wanted"], s["dy"])]


def _plain_norm(s):
    c, dt = s["case"], TYPES[s["case"]["type"]]
    f = lambda t: None if t is None else t.float()  # noqa: E731
    x, w, b = f(s["x"]), f(s["weight"]), f(s["bias"])
    x = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    xh = x * r
    y = xh if w is None else xh * w
    if b is not None:
        y = y + b
    y = y.to(dt)
    if c["pass"] == "apply":
        return y
    dy = s["dy"].float()
    gy = dy if w is None else dy * w
    out = [y, ((gy - gy.mean(1, keepdim=True) - xh * (gy * xh).mean(1, keepdim=True)) * r).to(dt)]
    if w is not None:
        out.append((dy * xh).sum(0).to(s["weight"].dtype))
    if b is not None:
        out.append(dy.sum(0).to(s["bias"].dtype))
    return out


def _act(z, act):
    """act(z) and its derivative."""
    if act == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if act == "silu":
        e = torch.sigmoid(z)
        return z * e, e * (1 + z * (1 - e))
    if act == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z * z * z))
        big, small = 0.5 + 0.5 * t, 0.5 * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    else:
        big = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        small = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z * big, big + z * small


def _plain_weight(s, name):
    """The float32 weight that the codes stand for."""
    c = s["case"]
    one = 2.0 ** (c["bits"] - 1)
    if c["pass"] == "serve":
        codes, scale = s[name]
        return codes.float() * (scale / one)[:, None]
    w = s[name].double()                              # a weight next to a border of two codes needs 64 bits
    top = w.abs().amax(1) if c["scale"] == "per_channel" else w.abs().amax().expand(c["n"])
    scale = torch.where(top > 0, top / torch.full_like(top, 1 - 1 / one), torch.ones_like(top)).float()
    return torch.round(w / scale.double()[:, None] * one).clamp(1 - one, one - 1).float() * (scale / one)[:, None]


def _plain_gated(s):
    c, dt = s["case"], TYPES[s["case"]["type"]]
    x, wg, wu = s["x"].float(), _plain_weight(s, "gate"), _plain_weight(s, "up")
    zg, zu = x @ wg.T, x @ wu.T
    if c["bias"]:
        zg, zu = zg + s["gate_bias"].float(), zu + s["up_bias"].float()
    a, slope = _act(zg, c["act"])
    h = (a * zu).to(dt)
    if c["pass"] == "serve":
        return h
    dh = s["dy"].float()
    dg, du = dh * zu * slope, dh * a
    out = [h, (dg @ wg + du @ wu).to(dt), (dg.T @ x).to(dt), (du.T @ x).to(dt)]
    return out + [dg.sum(0).to(dt), du.sum(0).to(dt)] if c["bias"] else out


def _plain_distill(s):
    c, dt, temp = s["case"], TYPES[s["case"]["type"]], s["case"]["temperature"]
    index = s["index"].clamp(min=0)
    there = s["index"] >= 0
    t = torch.where(there, s["teacher"].float() / temp, torch.full_like(index, -math.inf, dtype=torch.float32))
    some = there.any(1)
    t = torch.where(some[:, None], t, torch.zeros_like(t))
    t = t - t.amax(1, keepdim=True)
    e = torch.exp(t)
    total = e.sum(1, keepdim=True)
    p, logp = e / total * there, t - torch.log(total)
    z = s["logits"].float() / temp
    z = z - z.amax(1, keepdim=True)
    q = torch.exp(z)
    total = q.sum(1, keepdim=True)
    logq = z.gather(1, index) - torch.log(total)
    w = some.float() if s["mask"] is None else (some & s["mask"]).float()
    row = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(1) * (temp * temp) * w
    if c["reduction"] == "none":
        return row
    share = 1.0
    if c["reduction"] == "mean":
        share = w.sum()
        share = torch.where(share == 0, torch.zeros_like(share), 1 / share)
    loss = row.sum() * share
    if c["pass"] == "eval":
        return loss
    factor = (w * share * temp * s["dy"])[:, None]
    return [loss, (q / total * factor).scatter_add(1, index, -p * factor).to(dt)]


# --- what a pass cannot do without ----------------------------------------------------------------------------


def work(case):
    size, m = 4 if case["type"] == "f32" else 2, case["m"]
    train = case["pass"] == "train"
    if case["op"] == "norm":
        n, params = case["n"], {"both": 2, "weight": 1, "none": 0}[case["affine"]]
        each = params * n * (4 if case["params"] == "f32" else 2)
        return {"bytes": (4 if train else 2) * m * n * size + (2 if train else 1) * each, "flops": (16 if train else 7) * m * n}
    if case["op"] == "gated":
        k, n = case["k"], case["n"]
        extra = 2 * n * size if case["bias"] else 0
        if not train:
            return {"bytes": m * k * size + 2 * (n * k + 4 * n) + m * n * size + extra, "flops": 4 * m * n * k}
        return {"bytes": 2 * m * k * size + 4 * n * k * size + 2 * m * n * size + 2 * extra, "flops": 12 * m * n * k}
    v, k = case["v"], case["k"]
    teacher = m * k * (8 + (2 if case["type"] == "bf16" else 4)) + (m if case["mask"] else 0)
    return {"bytes": (2 if train else 1) * m * v * size + teacher, "flops": (7 if train else 4) * m * v}


# --- the definition in 64 bits --------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    out = {"norm": _exact_norm, "gated": _exact_gated, "distill": _exact_distill}[case["op"]](s)
    if case["pass"] != "train":
        return out.detach()
    result, inputs = out
    dy = s["dy"].double()
    return [result.detach(), *torch.autograd.grad(result, [t for t in inputs if t is not None], dy)]


def _leaf(t, train):
    return None if t is None else t.detach().double().requires_grad_(train)


def _exact_norm(s):
    train = s["case"]["pass"] == "train"
    x, w, b = (_leaf(s[name], train) for name in ("x", "weight", "bias"))
    y = torch.nn.functional.layer_norm(x, x.shape[1:], w, b, EPS)
    return (y, (x, w, b)) if train else y


def _exact_gated(s):
    c, fn = s["case"], torch.nn.functional
    train, unit = c["pass"] == "train", 2.0 ** (1 - c["bits"])
    x = _leaf(s["x"], train)
    inputs, z = [x], []
    for name in ("gate", "up"):
        if train:
            w = s[name].detach().double()
            per = w.abs().max(dim=1, keepdim=True).values if c["scale"] == "per_channel" else w.abs().max()
            per = torch.where(per > 0, per / (1 - unit), torch.ones_like(per)).float().double()
            weight = torch.round(w / (per * unit)).clamp(1 - 1 / unit, 1 / unit - 1) * unit * per
        else:
            weight = s[name][0].double() * unit * s[name][1].double().unsqueeze(1)
        inputs.append(_leaf(weight, train))
        z.append(fn.linear(x, inputs[-1]))
    for i, name in enumerate(("gate_bias", "up_bias")):
        inputs.append(_leaf(s[name], train))
        if s[name] is not None:
            z[i] = z[i] + inputs[-1]
    act = {"relu": fn.relu, "gelu": fn.gelu, "silu": fn.silu, "gelu_tanh": lambda v: fn.gelu(v, approximate="tanh")}
    h = act[c["act"]](z[0]) * z[1]
    return (h, inputs) if train else h


def _exact_distill(s):
    c, temp = s["case"], s["case"]["temperature"]
    train = c["pass"] == "train"
    logits = _leaf(s["logits"], train)
    logq = torch.log_softmax(logits / temp, dim=1)
    there = s["index"] >= 0
    counted = there.any(dim=1) if s["mask"] is None else there.any(dim=1) & s["mask"]
    logp = torch.log_softmax((s["teacher"].double() / temp).masked_fill(~there, -1e9), dim=1)
    near = torch.gather(logq, 1, s["index"].clamp(min=0))
    row = (logp.exp() * (logp - near)).masked_fill(~there, 0.0).sum(dim=1) * temp ** 2
    row = row.masked_fill(~counted, 0.0)
    if c["reduction"] == "none":
        return row
    loss = row.sum()
    if c["reduction"] == "mean":
        loss = loss / counted.sum().clamp(min=1)
    return (loss, [logits]) if train else loss
