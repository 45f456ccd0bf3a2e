"""The operators of deep residual trunks, as they are measured: norms around a block with its gate and residual scale
(forward, and forward + backward), 8-bit activation checkpoints (the packing itself, an activation and a Linear layer whose
backward passes read them).

`own = False` computes the plain form: elementary torch operations in 32 bits, rounded once at the end, gradients by autograd.
`own = True` makes the calls that a training program makes of scpair_amd.ops.  `exact` is the definition in 64 bits, with the
backward formulas written out.

The 8-bit form: every 64 columns of a row share a step 2^k, the smallest power of two with max|x| <= 127 * 2^k (and
k >= -126); the codes are x / 2^k rounded to the nearest whole number, ties to even, and a code c stands for c * 2^k.
"""
import math

import torch

own = False

GROUP = 64
MAX_NORM = 32768 * 4096            # elements of the largest norm / activation / packing case
MAX_LINEAR = 16384 * 4096 * 4096   # products of the largest Linear case


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _norm(name, rows, cols, x_type, h_type, train, post="layer", pre="layer", gate="none", gate_act="sigmoid",
          scale="column"):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "x_type": x_type, "h_type": h_type, "train": train,
            "post": post, "pre": pre, "gate": gate, "gate_act": gate_act, "scale": scale}


def listed():
    return [
        # one cell through one block of a trunk of the first hidden size, as at inference: latency counts
        _norm("norm_one_row", 1, 900, "float32", "float32", False),
        # a training minibatch of 1024 cells at that size, all in 32 bits, a gate for every element
        _norm("norm_train_fp32", 1024, 900, "float32", "float32", True, gate="full"),
        # residual stream in 32 bits beside blocks in bf16, batch of 4096
        _norm("norm_train_mixed", 4096, 2048, "float32", "bfloat16", True, post="rms", pre="rms", gate="full"),
        # odd width, the last minibatch of an epoch, one gate for each row, one learned residual scale
        _norm("norm_train_odd", 777, 4999, "bfloat16", "bfloat16", True, gate="row", gate_act="tanh", scale="scalar"),
        # large batch, wide trunk, a learned gate for every column
        _norm("norm_train_large", 32768, 4096, "bfloat16", "bfloat16", True, post="rms", pre="rms", gate="column"),
        # a checkpoint of the packed two-branch hidden layer of one minibatch, written and read back
        {"name": "pack_batch", "op": "pack", "rows": 1024, "cols": 1801, "type": "float32"},
        # the same of a large batch of a wide trunk
        {"name": "pack_large", "op": "pack", "rows": 16384, "cols": 8192, "type": "bfloat16"},
        # an activation of a minibatch, forward and backward
        {"name": "act_batch", "op": "act", "rows": 1024, "cols": 1801, "type": "float32", "kind": "gelu"},
        # the same of a large batch of a wide trunk
        {"name": "act_large", "op": "act", "rows": 16384, "cols": 8192, "type": "bfloat16", "kind": "silu"},
        # a Linear layer's training step between the hidden sizes, minibatch, 32 bits
        {"name": "linear_fp32", "op": "linear", "rows": 1024, "ins": 900, "outs": 1800, "type": "float32", "bias": True},
        # odd sizes in bf16
        {"name": "linear_odd", "op": "linear", "rows": 777, "ins": 1801, "outs": 901, "type": "bfloat16", "bias": True},
        # large batch, wide trunk
        {"name": "linear_large", "op": "linear", "rows": 16384, "ins": 4096, "outs": 4096, "type": "bfloat16",
         "bias": True},
    ]


def _log_size(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "pack", "act", "linear"])
    if op == "linear":
        case = {"op": op, "type": rng.choice(["float32", "bfloat16", "bfloat16"]), "bias": rng.random() < 0.8}
        top = MAX_LINEAR // (8 if case["type"] == "float32" else 1)
        case["ins"] = _log_size(rng, 8, 8192)
        case["outs"] = _log_size(rng, 8, 8192)
        case["rows"] = _log_size(rng, 1, min(16384, max(1, top // (case["ins"] * case["outs"]))))
        return case
    cols = _log_size(rng, 8, 8192)
    rows = _log_size(rng, 1, min(32768, MAX_NORM // cols))
    if op == "pack":
        return {"op": op, "rows": rows, "cols": cols, "type": rng.choice(["float32", "bfloat16"])}
    if op == "act":
        return {"op": op, "rows": rows, "cols": cols, "type": rng.choice(["float32", "bfloat16"]),
                "kind": rng.choice(["gelu", "silu", "leaky_relu"])}
    x_type, h_type = rng.choice([("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16")])
    case = _norm("", rows, cols, x_type, h_type, rng.random() < 0.75, post=rng.choice(["none", "rms", "layer"]),
                 pre=rng.choice(["rms", "layer"]), gate=rng.choice(["none", "full", "row", "column"]),
                 gate_act=rng.choice(["sigmoid", "tanh", "none"]), scale=rng.choice(["none", "scalar", "column"]))
    del case["name"]
    return case


def _bytes(type_name):
    return 4 if type_name == "float32" else 2


def work(case):
    if case["op"] == "linear":
        m, k, n, b = case["rows"], case["ins"], case["outs"], _bytes(case["type"])
        # in: x, W, dy (and b); out: y, dx, dW (and db)
        return {"bytes": b * 2 * (m * k + n * k + m * n) + (8 * n if case["bias"] else 0), "flops": 6 * m * n * k}
    n = case["rows"] * case["cols"]
    if case["op"] == "pack":
        b = _bytes(case["type"])
        return {"bytes": 2 * b * n + 2 * n + n // 32, "flops": 4 * n}       # x in, codes out and in, values out
    if case["op"] == "act":
        return {"bytes": 4 * _bytes(case["type"]) * n, "flops": 40 * n}     # in: z, da; out: a, dz
    bx, bh = _bytes(case["x_type"]), _bytes(case["h_type"])
    gate = {"none": 0, "full": n * bh, "row": 4 * case["rows"], "column": 4 * case["cols"]}[case["gate"]]
    if not case["train"]:
        return {"bytes": 2 * n * bx + 2 * n * bh + gate, "flops": 16 * n}   # in: x, h; out: r, y
    return {"bytes": 4 * n * bx + 4 * n * bh + 2 * gate, "flops": 60 * n}   # and dr, dy; dx, dh


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g, rows, cols, dtype):
    """Values as hidden layers have them: columns of different spread, a few of them large, some rows louder."""
    t = _randn(g, rows, cols)
    spread = torch.exp(0.3 * _randn(g, cols))
    spread = torch.where(torch.rand((cols,), generator=g, device="cuda") < 0.01, 8.0 * spread, spread)
    t.mul_(spread).mul_(torch.exp(0.2 * _randn(g, rows, 1))).add_(0.1)
    return t.to(dtype)


def _type(name):
    return torch.float32 if name == "float32" else torch.bfloat16


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "linear":
        m, k, n, t = case["rows"], case["ins"], case["outs"], _type(case["type"])
        s["x"] = _activations(g, m, k, t).requires_grad_()
        s["W"] = (_randn(g, n, k) / math.sqrt(k)).to(t).requires_grad_()
        s["b"] = (0.1 * _randn(g, n)).requires_grad_() if case["bias"] else None
        s["dy"] = (1e-2 * _randn(g, m, n)).to(t)
        return s
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "pack":
        s["x"] = _activations(g, rows, cols, _type(case["type"]))
        return s
    if case["op"] == "act":
        s["z"] = _activations(g, rows, cols, _type(case["type"])).requires_grad_()
        s["da"] = (1e-2 * _randn(g, rows, cols)).to(_type(case["type"]))
        return s
    tx, th = _type(case["x_type"]), _type(case["h_type"])
    train = case["train"]
    s["x"] = _activations(g, rows, cols, tx).requires_grad_(train)
    s["h"] = _activations(g, rows, cols, th).requires_grad_(train)
    gate = {"none": None, "full": (rows, cols), "row": (rows, 1), "column": (cols,)}[case["gate"]]
    if gate is not None:
        gate = _randn(g, *gate)
        gate = (gate.to(th) if case["gate"] == "full" else gate).requires_grad_(train)
    s["gate"] = gate
    scale = {"none": None, "scalar": (1,), "column": (cols,)}[case["scale"]]
    s["scale"] = None if scale is None else (0.5 + 0.1 * _randn(g, *scale)).requires_grad_(train)
    for norm in ("post", "pre"):
        kind = case[norm]
        s[norm + "_weight"] = None if kind == "none" else (1.0 + 0.1 * _randn(g, cols)).requires_grad_(train)
        s[norm + "_bias"] = (0.1 * _randn(g, cols)).requires_grad_(train) if kind == "layer" else None
    if train:
        s["dr"] = (1e-2 * _randn(g, rows, cols)).to(tx)
        s["dy"] = (1e-2 * _randn(g, rows, cols)).to(th)
    return s


_NORM_LEAVES = ("x", "h", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _checkpoint_plain(x):
    """The values that the 8-bit form of x stands for, in 32 bits."""
    rows, cols = x.shape
    pad = (-cols) % GROUP
    t = x.float()
    if pad:
        t = torch.cat([t, t.new_zeros(rows, pad)], 1)
    t = t.reshape(rows, -1, GROUP)
    m, e = torch.frexp(t.abs().amax(2, keepdim=True))
    k = torch.where(m <= 127.0 / 128.0, e - 7, e - 6).clamp(min=-126)
    step = ((127 + k) << 23).to(torch.int32).view(torch.float32)
    inverse = ((127 - k) << 23).to(torch.int32).view(torch.float32)
    return (torch.round(t * inverse) * step).reshape(rows, -1)[:, :cols]


def _norm_plain(t, kind, weight, bias):
    if kind == "none":
        return t
    if kind == "rms":
        return t * torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-5) * weight
    c = t - t.mean(1, keepdim=True)
    return c * torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5) * weight + bias


def _run_norm_plain(s):
    case = s["case"]
    u = _norm_plain(s["h"].float(), case["post"], s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        gate = s["gate"].float()
        u = u * {"sigmoid": torch.sigmoid, "tanh": torch.tanh, "none": lambda v: v}[case["gate_act"]](gate)
    if s["scale"] is not None:
        u = u * s["scale"]
    r = s["x"].float() + u
    y = _norm_plain(r, case["pre"], s["pre_weight"], s["pre_bias"])
    return r.to(s["x"].dtype), y.to(s["h"].dtype)


class _PlainAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, kind):
        ctx.save_for_backward(_checkpoint_plain(z))
        ctx.kind = kind
        t = z.float()
        if kind == "gelu":
            a = 0.5 * t * (1.0 + torch.erf(t * math.sqrt(0.5)))
        elif kind == "silu":
            a = t / (1.0 + torch.exp(-t))
        else:
            a = torch.where(t > 0, t, 0.01 * t)
        return a.to(z.dtype)

    @staticmethod
    def backward(ctx, da):
        v, = ctx.saved_tensors
        if ctx.kind == "gelu":
            slope = 0.5 * (1.0 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
        elif ctx.kind == "silu":
            sig = 1.0 / (1.0 + torch.exp(-v))
            slope = sig * (1.0 + v * (1.0 - sig))
        else:
            slope = torch.where(v > 0, 1.0, 0.01)
        return (da.float() * slope).to(da.dtype), None


class _PlainLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W, b):
        ctx.save_for_backward(_checkpoint_plain(x), W)
        y = x.float() @ W.float().t()
        return (y if b is None else y + b).to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        v, W = ctx.saved_tensors
        d = dy.float()
        return (d @ W.float()).to(dy.dtype), (d.t() @ v).to(W.dtype), d.sum(0) if ctx.needs_input_grad[2] else None


def run(state):
    case = state["case"]
    if own:
        from scpair_amd import ops
    if case["op"] == "pack":
        x = state["x"]
        return ops.unpack8(ops.pack8(x)) if own else _checkpoint_plain(x).to(x.dtype)
    if case["op"] == "act":
        z = state["z"]
        a = ops.act8(z, case["kind"]) if own else _PlainAct.apply(z, case["kind"])
        return a, torch.autograd.grad(a, z, state["da"])[0]
    if case["op"] == "linear":
        x, W, b = state["x"], state["W"], state["b"]
        y = ops.linear8(x, W, b) if own else _PlainLinear.apply(x, W, b)
        return (y,) + torch.autograd.grad(y, [t for t in (x, W, b) if t is not None], state["dy"])
    if own:
        r, y = ops.gated_residual_norm(
            state["x"], state["h"], gate=state["gate"], gate_act=case["gate_act"], scale=state["scale"],
            post=None if case["post"] == "none" else case["post"], post_weight=state["post_weight"],
            post_bias=state["post_bias"], pre=case["pre"], pre_weight=state["pre_weight"], pre_bias=state["pre_bias"],
            eps=1e-5)
    else:
        r, y = _run_norm_plain(state)
    if not case["train"]:
        return r, y
    leaves = [state[n] for n in _NORM_LEAVES if state[n] is not None]
    return (r, y) + torch.autograd.grad((r, y), leaves, (state["dr"], state["dy"]))


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _checkpoint_exact(x):
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[1], GROUP):
        part = x[:, c:c + GROUP].double()
        top = part.abs().max(1, keepdim=True).values
        # smallest k >= -126 with top <= 127 * 2^k, from a first guess that is off by one at most
        k = (torch.floor(torch.log2(top.clamp(min=2.0 ** -149))) - 7).clamp(min=-126).long()
        for _ in range(3):
            k = torch.where(top > 127.0 * _power(k), k + 1, k)
        out[:, c:c + GROUP] = torch.round(part / _power(k)) * _power(k)
    return out


def _power(k):
    return ((k + 1023) << 52).view(torch.float64)


def _norm_exact(t, kind, weight, bias):
    """normalised values, 1 / spread, and the result"""
    if kind == "none":
        return None, None, t
    mean = t.mean(1, keepdim=True) if kind == "layer" else 0.0
    inv = 1.0 / torch.sqrt(((t - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    hat = (t - mean) * inv
    return hat, inv, hat * weight.double() + (bias.double() if bias is not None else 0.0)


def _norm_exact_backward(d, hat, inv, kind, weight):
    """gradient of the norm's input; of its weight; of its bias"""
    if kind == "none":
        return d, None, None
    a = d * weight.double()
    back = a - hat * (a * hat).mean(1, keepdim=True)
    if kind == "layer":
        back = back - a.mean(1, keepdim=True)
    return inv * back, (d * hat).sum(0), d.sum(0) if kind == "layer" else None


def exact(case, seed):
    s = prepare(case, seed)
    s = {n: (t.detach() if isinstance(t, torch.Tensor) else t) for n, t in s.items()}
    if case["op"] == "pack":
        return _checkpoint_exact(s["x"])
    if case["op"] == "act":
        t, v, d = s["z"].double(), _checkpoint_exact(s["z"]), s["da"].double()
        if case["kind"] == "gelu":
            return t * torch.special.ndtr(t), d * (torch.special.ndtr(v)
                                                   + v * torch.exp(-v * v / 2) * (2 * math.pi) ** -0.5)
        if case["kind"] == "silu":
            f = torch.sigmoid(v)
            return t * torch.sigmoid(t), d * (f + v * f * torch.sigmoid(-v))
        return t * (0.01 + 0.99 * (t > 0)), d * (0.01 + 0.99 * (v > 0))
    if case["op"] == "linear":
        x, W, d = s["x"].double(), s["W"].double(), s["dy"].double()
        y = x @ W.t()
        if s["b"] is not None:
            y = y + s["b"].double()
        grads = [d @ W, d.t() @ _checkpoint_exact(s["x"])] + ([d.sum(0)] if s["b"] is not None else [])
        return (y, *grads)
    x, h = s["x"].double(), s["h"].double()
    hat1, inv1, n = _norm_exact(h, case["post"], s["post_weight"], s["post_bias"])
    raw = s["gate"].double() if s["gate"] is not None else None
    if raw is None:
        g, g1 = 1.0, None
    elif case["gate_act"] == "sigmoid":
        g = torch.sigmoid(raw)
        g1 = g * torch.sigmoid(-raw)
    elif case["gate_act"] == "tanh":
        g = torch.tanh(raw)
        g1 = 1.0 / torch.cosh(raw) ** 2
    else:
        g, g1 = raw, torch.ones_like(raw)
    sc = s["scale"].double() if s["scale"] is not None else 1.0
    r = x + sc * g * n
    hat2, inv2, y = _norm_exact(r, case["pre"], s["pre_weight"], s["pre_bias"])
    if not case["train"]:
        return r, y
    back, dw2, db2 = _norm_exact_backward(s["dy"].double(), hat2, inv2, case["pre"], s["pre_weight"])
    du = s["dr"].double() + back
    dgate = dscale = None
    if raw is not None:
        dgate = du * sc * n * g1
        if case["gate"] == "row":
            dgate = dgate.sum(1, keepdim=True)
        elif case["gate"] == "column":
            dgate = dgate.sum(0)
    if s["scale"] is not None:
        dscale = (du * g * n).sum(0)
        if case["scale"] == "scalar":
            dscale = dscale.sum().reshape(1)
    dh, dw1, db1 = _norm_exact_backward(du * sc * g, hat1, inv1, case["post"], s["post_weight"])
    grads = {"x": du, "h": dh, "gate": dgate, "scale": dscale, "post_weight": dw1, "post_bias": db1,
             "pre_weight": dw2, "pre_bias": db2}
    return (r, y) + tuple(grads[n] for n in _NORM_LEAVES if s[n] is not None)
