"""The cases on which the tensor-core linear over sf codes and the multi-tensor AdamW step are measured.

``run`` computes an operator either in its plain form (elementary torch operations in 32 bits, 64 where a value stands
next to a border) or, where ``own`` is true, through the package's public calls.  Both get the same state.

linear   y = act(x Wq^T + b) + r,  Wq[n, k] = code[n, k] 2^-(bits-1) scale[n].
         pass "serve": the codes and scales are at hand (a packed weight);
         pass "train": the float weight is quantized in the pass, and the pass returns y and the gradients of x,
         the weight (straight through), the bias and the residual.
adamw    one step over a list of tensors, the moments in float32 or in sf8 blocks of 256.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
BLOCK = 256                       # elements that share one scale in an sf8 moment
SMALL = 4096                      # tensors below this keep float32 moments beside sf8 ones
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01

# the tensors of a GPT-2-small embedding and one of its blocks (vocabulary 50257, width 768, 1024 positions)
GPT2 = "38597376,786432,768,768,1769472,2304,589824,768,768,768,2359296,2359296,768"


def listed():
    return [
        # one token of a served model, a square projection: bound by the weight's bytes and the latency of the call
        {"name": "serve one token", "op": "linear", "pass": "serve", "m": 1, "k": 4096, "n": 4096, "type": "bf16",
         "bits": 8, "act": "silu", "bias": True, "residual": False, "pad": 0},
        # a few sequences decoded together through an LM head: an odd vocabulary, an odd number of rows
        {"name": "serve head of 13", "op": "linear", "pass": "serve", "m": 13, "k": 768, "n": 50257, "type": "fp16",
         "bits": 8, "act": "none", "bias": False, "residual": False, "pad": 0},
        # a prompt: bound by the tensor cores
        {"name": "serve prompt", "op": "linear", "pass": "serve", "m": 4096, "k": 4096, "n": 8192, "type": "bf16",
         "bits": 8, "act": "gelu", "bias": True, "residual": True, "pad": 0},
        # a ragged prompt through odd sizes, sf6 codes, rows of a wider buffer
        {"name": "serve odd", "op": "linear", "pass": "serve", "m": 777, "k": 1031, "n": 2049, "type": "fp16",
         "bits": 6, "act": "relu", "bias": True, "residual": True, "pad": 5},
        # fine-tuning the attention projection of a converted GPT-2-small on 8 x 512 tokens
        {"name": "train projection", "op": "linear", "pass": "train", "m": 4096, "k": 768, "n": 2304, "type": "bf16",
         "bits": 8, "act": "gelu_tanh", "bias": True, "residual": False, "pad": 0, "scale": "per_channel"},
        # fine-tuning a wide layer with its residual
        {"name": "train wide", "op": "linear", "pass": "train", "m": 8192, "k": 4096, "n": 4096, "type": "fp16",
         "bits": 8, "act": "silu", "bias": True, "residual": True, "pad": 0, "scale": "per_tensor"},
        # a few small tensors (an adapter's): bound by the latency of the call
        {"name": "adamw adapter", "op": "adamw", "sizes": "6144,6144,768,1001,36864,7", "type": "f32",
         "state": "f32"},
        # an embedding and a block of GPT-2-small, float32 states
        {"name": "adamw f32", "op": "adamw", "sizes": GPT2, "type": "f32", "state": "f32"},
        # the same with sf8 states
        {"name": "adamw sf8", "op": "adamw", "sizes": GPT2, "type": "f32", "state": "sf8"},
        # the layers of a wide model kept in bf16, sf8 states
        {"name": "adamw sf8 bf16", "op": "adamw", "sizes": "16777216,16777216,33554432,33554432,4096,4096,12345679",
         "type": "bf16", "state": "sf8"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["serve", "serve", "train", "adamw"])
    if kind == "adamw":
        left, sizes = 1 << 26, []
        for _ in range(rng.randint(1, 16)):
            n = _log(rng, 1, 1 << 24)
            if n <= left:
                sizes.append(n)
                left -= n
        return {"op": "adamw", "sizes": ",".join(map(str, sizes)), "type": rng.choice(["f32", "bf16", "fp16"]),
                "state": rng.choice(["f32", "sf8", "sf8"])}
    c = {"op": "linear", "pass": kind, "m": _log(rng, 1, 4096), "k": _log(rng, 16, 4096), "n": _log(rng, 16, 8192),
         "type": rng.choice(["bf16", "fp16"]), "bits": rng.choice([4, 5, 6, 7, 8, 8, 8]),
         "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.7,
         "residual": rng.random() < 0.4, "pad": rng.choice([0, 0, 1, 8])}
    if rng.random() < 0.5:                            # half of the cases are aligned as layers mostly are
        c["k"], c["n"] = 16 * max(1, c["k"] // 16), 16 * max(1, c["n"] // 16)
    if kind == "train":
        c["scale"] = rng.choice(["per_tensor", "per_channel"])
    return c


# --- inputs ---------------------------------------------------------------------------------------------------


def _sizes(case):
    return [int(s) for s in case["sizes"].split(",")]


def _blocks(t):
    """A flat tensor as rows of BLOCK, the last one filled with zeros."""
    return torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)).view(-1, BLOCK)


def _first_moments(g, n, power, size):
    """sf8 codes and scales as a run of steps leaves them: the moment (a normal value to `power`) companded."""
    z = torch.randn(n, generator=g, device="cuda").abs_().pow_(power)
    b = _blocks(z)
    top = b.amax(1)
    code = (127 * (b / top[:, None]).pow(0.5 / power)).round_().view(-1)[:n].clamp_(min=1)
    if power == 1:
        code = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, -code, code)
    return code.to(torch.int8), top * size


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    dt = TYPES[case["type"]]
    if case["op"] == "adamw":
        s = {"case": case, "step": 10, "p": [], "g": [], "m": [], "v": []}
        for n in _sizes(case):
            s["p"].append(normal(n, std=0.02, dtype=dt))
            s["g"].append(normal(n, std=1e-2, dtype=dt))
            if case["state"] == "sf8" and n >= SMALL:
                s["m"].append(_first_moments(g, n, 1, 1e-3))
                s["v"].append(_first_moments(g, n, 2, 1e-4))
            else:
                s["m"].append(normal(n, std=1e-3))
                s["v"].append(normal(n, std=1e-2).square_())
        return s
    m, k, n = case["m"], case["k"], case["n"]
    s = {"case": case, "x": normal(m, k + case["pad"], dtype=dt)[:, :k]}
    w = normal(n, k, std=k ** -0.5, dtype=dt)
    s["bias"] = normal(n, std=0.1, dtype=dt) if case["bias"] else None
    s["residual"] = normal(m, n, dtype=dt) if case["residual"] else None
    if case["pass"] == "serve":
        s["scale"] = (w.float().abs().amax(1) / _largest(case)).clamp_(min=1e-20)
        s["codes"] = torch.round(w.float() / s["scale"][:, None] * 2.0 ** (case["bits"] - 1)).clamp_(
            1 - 2 ** (case["bits"] - 1), 2 ** (case["bits"] - 1) - 1).to(torch.int8)
    else:
        s["weight"] = w.requires_grad_()
        s["dy"] = normal(m, n, dtype=dt)
        for name in ("x", "bias", "residual"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def _largest(case):
    """The largest value of the sf format: M / 2^(bits-1)."""
    return 1.0 - 2.0 ** (1 - case["bits"])


# --- one pass -------------------------------------------------------------------------------------------------


def run(state):
    if own:
        return _own_adamw(state) if state["case"]["op"] == "adamw" else _own_linear(state)
    return _plain_adamw(state) if state["case"]["op"] == "adamw" else _plain_linear(state)


def _own_linear(s):
    import superfloat.python_b200.torch as sft
    c = s["case"]
    act = None if c["act"] == "none" else c["act"]
    if c["pass"] == "serve":
        w = sft.SFPackedWeight(s["codes"], s["scale"], c["bits"])
        return sft.tensor_linear(s["x"], w, s["bias"], activation=act, residual=s["residual"])
    y = sft.tensor_linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"],
                          dtype="sf%d" % c["bits"], scale=c["scale"])
    wanted = [t for t in (s["x"], s["weight"], s["bias"], s["residual"]) if t is not None]
    return [y, *torch.autograd.grad(y, wanted, s["dy"])]


def _own_adamw(s):
    import superfloat.python_b200.torch as sft
    s["step"] += 1
    m, v = ([sft.SF8Moment(*t) if isinstance(t, tuple) else t for t in s[name]] for name in ("m", "v"))
    sft.adamw_step(s["p"], s["g"], m, v, step=s["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                   dither=s["step"])
    return [s["p"], sft.moment_values(m, "first"), sft.moment_values(v, "second")]


def _gelu_parts(z, tanh):
    """(Phi, phi) of gelu(z) = z Phi(z), gelu'(z) = Phi(z) + z phi(z); of the tanh form likewise."""
    if tanh:
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 + 0.5 * t, 0.5 * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))), torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _act(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if act == "silu":
        e = torch.sigmoid(z)
        return z * e, e * (1 + z * (1 - e))
    big, small = _gelu_parts(z, act == "gelu_tanh")
    return z * big, big + z * small


def _plain_linear(s):
    c = s["case"]
    one = 2.0 ** (c["bits"] - 1)
    f = lambda t: None if t is None else t.detach().float()  # noqa: E731
    x, bias, res = f(s["x"]), f(s["bias"]), f(s["residual"])
    if c["pass"] == "serve":
        wq = s["codes"].float() * (s["scale"] / one)[:, None]
    else:
        w = s["weight"].detach().double()             # a weight next to a border of two codes needs 64 bits
        top = w.abs().amax(1) if c["scale"] == "per_channel" else w.abs().amax().expand(c["n"])
        scale = torch.where(top > 0, top / torch.full_like(top, _largest(c)), torch.ones_like(top)).float()
        wq = (torch.round(w / scale.double()[:, None] * one).clamp(1 - one, one - 1)).float() * (scale / one)[:, None]
    z = x @ wq.T
    if bias is not None:
        z = z + bias
    y, d = _act(z, c["act"])
    if res is not None:
        y = y + res
    dt = TYPES[c["type"]]
    y = y.to(dt)
    if c["pass"] == "serve":
        return y
    dz = s["dy"].float() * d
    out = [y, (dz @ wq).to(dt), (dz.T @ x).to(dt)]
    if bias is not None:
        out.append(dz.sum(0).to(dt))
    if res is not None:
        out.append(s["dy"])
    return out


def _dither(n, seed):
    """Two uniform 16-bit numbers for each of n elements: a counter mixed to 32 bits."""
    low = 0xFFFFFFFF
    h = (torch.arange(n, device="cuda") * 0x9E3779B1 + seed) & low
    h = h ^ (h >> 16)
    h = (h * 0x7FEB352D) & low
    h = h ^ (h >> 15)
    h = (h * 0x846CA68B) & low
    h = h ^ (h >> 16)
    return (h & 0xFFFF).float() * 2.0 ** -16, (h >> 16).float() * 2.0 ** -16


def _levels(c, power):
    c2 = c * c
    return c2 if power == 2 else c2 * c2


def _moment(code, scale, power):
    """The values that sf8 codes stand for: sign s (|c| / 127)^power."""
    c = code.float()
    unit = scale * (1.0 / 127.0 ** power)
    mag = _levels(c.abs(), power) * unit.repeat_interleave(BLOCK)[: code.numel()]
    return torch.where(c < 0, -mag, mag)


def _code(value, u, power):
    """Codes and scales of new moments: the two levels around a value, the upper one where the dither is below
    its share of the step.  A block whose largest moment is under 1e-30 is held as zero; a positive second
    moment keeps a code of at least one."""
    n = value.numel()
    top = _blocks(value.abs()).amax(1)
    top = torch.where(top < 1e-30, torch.zeros_like(top), top)
    inv = torch.where(top > 0, torch.full_like(top, 127.0 ** power) / top, torch.zeros_like(top))
    t = value.abs() * inv.repeat_interleave(BLOCK)[:n]
    c = torch.sqrt(t) if power == 2 else torch.sqrt(torch.sqrt(t))
    c = torch.floor(c)
    c = torch.where(_levels(c, power) > t, c - 1, c)
    c = torch.where(_levels(c + 1, power) <= t, c + 1, c).clamp(0, 127)
    low = _levels(c, power)
    up = (u * (_levels(c + 1, power) - low) < t - low) & (c < 127)
    c = c + up
    if power == 4:
        c = torch.where((t > 0) & (c == 0), torch.ones_like(c), c)
    return torch.where(value < 0, -c, c).to(torch.int8), top


def _plain_adamw(s):
    s["step"] += 1
    (b1, b2), t = BETAS, s["step"]
    shrink, size, root = 1 - LR * DECAY, LR / (1 - b1 ** t), 1 / math.sqrt(1 - b2 ** t)

    def one(i):
        p, g, m, v = s["p"][i], s["g"][i].float(), s["m"][i], s["v"][i]
        eight = isinstance(m, tuple)
        m0, v0 = (_moment(*m, 2), _moment(*v, 4)) if eight else (m, v)
        m1 = m0 * b1 + g * (1 - b1)
        v1 = v0 * b2 + (g * (1 - b2)) * g
        p.copy_(p.float() * shrink - m1 / (torch.sqrt(v1) * root + EPS) * size)
        if not eight:
            m.copy_(m1)
            v.copy_(v1)
            return p, m, v
        um, uv = _dither(p.numel(), (t + i * 0x9E3779B9) & 0xFFFFFFFF)
        for old, new in zip(m + v, _code(m1, um, 2) + _code(v1, uv, 4)):
            old.copy_(new)
        return p, _moment(*m, 2), _moment(*v, 4)

    p, m, v = zip(*[one(i) for i in range(len(s["p"]))])
    return [list(p), list(m), list(v)]


# --- what a pass cannot do without ----------------------------------------------------------------------------


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "adamw":
        bytes_ = 0
        for n in _sizes(case):
            bytes_ += 3 * size * n                    # the parameter read and written, the gradient read
            if case["state"] == "sf8" and n >= SMALL:
                # codes and scales read and written, and the values that they stand for returned
                bytes_ += 2 * (2 * n + 2 * 4 * -(-n // BLOCK)) + 2 * 4 * n
            else:
                bytes_ += 2 * 8 * n
        return {"bytes": bytes_, "flops": 12 * sum(_sizes(case))}
    m, k, n = case["m"], case["k"], case["n"]
    out = m * n * size
    extra = (n * size if case["bias"] else 0) + (out if case["residual"] else 0)
    if case["pass"] == "serve":
        return {"bytes": m * k * size + n * k + 4 * n + out + extra, "flops": 2 * m * n * k}
    return {"bytes": 2 * m * k * size + 2 * n * k * size + 2 * out + extra + (n * size if case["bias"] else 0),
            "flops": 6 * m * n * k}


# --- the definition in 64 bits --------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_adamw(s) if case["op"] == "adamw" else _exact_linear(s)


def _exact_linear(s):
    c = s["case"]
    unit = 2.0 ** (1 - c["bits"])
    with torch.no_grad():
        if c["pass"] == "serve":
            weight = s["codes"].double() * unit * s["scale"].double().unsqueeze(1)
        else:
            w = s["weight"].double()
            per = w.abs().max(dim=1, keepdim=True).values if c["scale"] == "per_channel" else w.abs().max()
            per = torch.where(per > 0, per / (1 - unit), torch.ones_like(per)).float().double()
            weight = torch.round(w / (per * unit)).clamp(1 - 1 / unit, 1 / unit - 1) * unit * per
        pre = torch.nn.functional.linear(s["x"].double(), weight, None if s["bias"] is None else s["bias"].double())
    pre.requires_grad_(c["pass"] == "train")
    fn = torch.nn.functional
    y = {"none": lambda v: v * 1.0, "relu": fn.relu, "gelu": fn.gelu, "silu": fn.silu,
         "gelu_tanh": lambda v: fn.gelu(v, approximate="tanh")}[c["act"]](pre)
    out = y.detach() if s["residual"] is None else y.detach() + s["residual"].detach().double()
    if c["pass"] == "serve":
        return out
    dz, = torch.autograd.grad(y, pre, s["dy"].double())
    got = [out, dz.mm(weight), torch.mm(dz.t(), s["x"].detach().double())]
    if s["bias"] is not None:
        got.append(dz.sum(dim=0))
    if s["residual"] is not None:
        got.append(s["dy"].double())
    return got


def _exact_adamw(s):
    """Parameters and float32 moments.  An sf8 moment has no value in 64 bits: where the float32 moment stands
    on a border of two codes, its last bit decides which one is kept."""
    s["step"] += 1
    b1, b2 = BETAS
    rise1, rise2 = 1 - b1 ** s["step"], 1 - b2 ** s["step"]

    def value(t, power):
        if not isinstance(t, tuple):
            return t.double()
        code, scale = t
        part = code.double() / 127
        at = torch.arange(code.numel(), device="cuda") // BLOCK
        return part.sign() * part.abs() ** power * scale.double()[at]

    p, m, v = [], [], []
    for p0, g, m0, v0 in zip(s["p"], s["g"], s["m"], s["v"]):
        g = g.double()
        m1 = torch.lerp(g, value(m0, 2), b1)
        v1 = torch.lerp(g.square(), value(v0, 4), b2)
        eight = isinstance(m0, tuple)
        p.append(p0.double() * (1 - LR * DECAY) - LR * (m1 / rise1) / ((v1 / rise2).sqrt() + EPS))
        m.append(None if eight else m1)
        v.append(None if eight else v1)
    return [p, m, v]
