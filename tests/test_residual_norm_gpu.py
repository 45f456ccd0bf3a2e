"""ops.gated_residual_norm (csrc/residual_norm.hip) against its definition in 64 bits on the CPU, gradients by autograd
there, over types, norms, gates, widths of every kernel variant, odd sizes and strides.

Tolerances.  An output held in bf16 is off by at most half a step, 2^-8 relative, of a value that carries the fp32 error.
fp32 error: every element is a chain of some 12 fp32 operations on values bounded by the row's largest terms; the row sums
of D terms add at most log2(D) + 32 roundings of their absolute terms.  With e = 2^-24 that is below 64 e relative to the
largest absolute value of the row's terms, which the test bounds by the tensor's own largest absolute value M of that
output (M >= the terms' scale for these inputs, condition numbers of order 1): |error| <= 128 e M for elements.  Column sums
of N terms accumulate N / 512 + 40 roundings of terms up to the largest |term|: |error| <= (N / 512 + 128) e * sum |term|, with
sum |term| bounded by N times the largest upstream gradient times the largest factor; the test takes the sum of absolute
terms from the oracle (gradients of the absolute problem) as sqrt(N) * M * 8, since terms of random sign add to M ~ sqrt(N)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, B16 = torch.float32, torch.bfloat16
NAMES = ("x", "h", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")


def _norm(t, kind, w, b, eps):
    if kind is None:
        return t
    c = t - t.mean(-1, keepdim=True) if kind == "layer" else t
    n = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    if w is not None:
        n = n * w
    return n if b is None else n + b


def oracle(t, post, pre, act, eps):
    """t: dict of float64 CPU tensors or None"""
    x, h = t["x"], t["h"]
    if h is None:
        r = x
    else:
        u = _norm(h, post, t["post_weight"], t["post_bias"], eps)
        if t["gate"] is not None:
            u = u * {"sigmoid": torch.sigmoid, "tanh": torch.tanh, "none": lambda v: v}[act](t["gate"])
        if t["scale"] is not None:
            u = u * t["scale"]
        r = x + u
    return r, _norm(r, pre, t["pre_weight"], t["pre_bias"], eps)


def inputs(shape, xt, ht, post, pre, gate, scale, seed, with_h=True):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    rn = lambda *s: torch.randn(*s, generator=g)
    t = dict.fromkeys(NAMES)
    t["x"] = (rn(*shape) + 0.2).to(xt)
    if with_h:
        t["h"] = (1.5 * rn(*shape) - 0.3).to(ht)
        t["gate"] = {None: None, "full": rn(*shape).to(ht), "row": rn(*shape[:-1], 1), "col": rn(D)}[gate]
        t["scale"] = {None: None, "one": 0.5 + 0.1 * rn(1), "col": 0.5 + 0.1 * rn(D)}[scale]
        if post is not None:
            t["post_weight"] = 1 + 0.1 * rn(D)
            t["post_bias"] = 0.1 * rn(D) if post == "layer" else None
    t["pre_weight"] = 1 + 0.1 * rn(D)
    t["pre_bias"] = 0.1 * rn(D) if pre == "layer" else None
    t["dr"], t["dy"] = rn(*shape).to(xt), rn(*shape).to(ht)
    return t


def kwargs(t, post, pre, act, eps):
    return dict(gate=t["gate"], scale=t["scale"], post=post, post_weight=t["post_weight"], post_bias=t["post_bias"], pre=pre,
                pre_weight=t["pre_weight"], pre_bias=t["pre_bias"], gate_act=act, eps=eps)


def close(name, got, want, rows, summed, dtype):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    M = want.abs().max().item()
    e = 2.0 ** -24
    tol = (rows / 512 + 128) * e * math.sqrt(rows) * 8 * max(M, 1.0) if summed else 128 * e * max(M, 1.0)
    bound = tol + (want.abs() * 2.0 ** -8 if dtype == B16 else 0.0)
    bad = (got - want).abs() - bound
    assert bad.max().item() <= 0, f"{name}: error {(got - want).abs().max().item()} (largest value {M}, tolerance {tol})"


def check(t, post, pre, act, eps=1e-5, use_dr=True, use_dy=True, layout=lambda v: v):
    from scpair_amd import ops
    dev = torch.device("cuda:0")
    ref = {n: None if t[n] is None else t[n].double().requires_grad_() for n in NAMES}
    r, y = oracle(ref, post, pre, act, eps)
    mine = {n: None if t[n] is None else layout(t[n].to(dev)).requires_grad_() for n in NAMES}
    gr, gy = ops.gated_residual_norm(mine["x"], mine["h"], **kwargs(mine, post, pre, act, eps))
    rows = t["x"].numel() // t["x"].shape[-1]
    xt, ht = t["x"].dtype, t["dy"].dtype
    if t["h"] is None:
        assert gr is mine["x"]
    close("r", gr, r.detach(), rows, False, xt)
    close("y", gy, y.detach(), rows, False, ht)
    assert gr.dtype == xt and gy.dtype == (ht if t["h"] is not None else xt)
    outs, gouts, ups, gups = [], [], [], []
    if use_dr:
        outs.append(r); gouts.append(gr); ups.append(t["dr"].double()); gups.append(layout(t["dr"].to(dev)))
    if use_dy:
        outs.append(y); gouts.append(gy); ups.append(t["dy"].double()); gups.append(layout(t["dy"].to(dev)))
    names = [n for n in NAMES if t[n] is not None]
    want = torch.autograd.grad(outs, [ref[n] for n in names], ups, allow_unused=True)
    got = torch.autograd.grad(gouts, [mine[n] for n in names], gups, allow_unused=True)
    again = None
    for n, g, w in zip(names, got, want):
        if w is None:
            assert g is None or not g.abs().any()
            continue
        summed = n not in ("x", "h") and not (n == "gate" and g.shape == t["x"].shape)
        # a row gate's gradient is a sum over the row's columns
        k = t["x"].shape[-1] if n == "gate" and g.shape[-1:] == (1,) and t["x"].shape[-1] > 1 else rows
        if n == "scale" and g.numel() == 1:
            k = t["x"].numel()
        close("d" + n, g, w, k, summed, t[n].dtype)
        assert g.dtype == t[n].dtype
    return gr, gy, got


TYPES = [(F32, F32), (F32, B16), (B16, B16)]
# widths of every variant: below a chunk, odd, 8 to 64 lanes to a row, workgroups of 2 to 16 waves with one and two chunks
WIDTHS = [1, 7, 8, 30, 64, 65, 128, 129, 256, 257, 511, 512, 513, 900, 1024, 1025, 2047, 2048, 2500, 4096, 4099, 6145, 8192, 8193, 16383,
          16384]


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("types", TYPES, ids=["f32", "mixed", "bf16"])
def test_widths(cols, types):
    # D = 1 under 'layer' is a row without spread: its gradient is exactly zero up to the rounding of the mean
    t = inputs((13, cols), *types, "layer" if cols > 1 else "rms", "rms", "full", "col", seed=cols)
    check(t, "layer" if cols > 1 else "rms", "rms", "sigmoid")
    t = inputs((5, cols), *types, "rms", "layer" if cols > 1 else "rms", "col", "one", seed=cols + 1)
    check(t, "rms", "layer" if cols > 1 else "rms", "tanh")


@pytest.mark.parametrize("post", [None, "rms", "layer"])
@pytest.mark.parametrize("pre", ["rms", "layer"])
@pytest.mark.parametrize("gate", [None, "full", "row", "col"])
@pytest.mark.parametrize("scale", [None, "one", "col"])
def test_forms(post, pre, gate, scale):
    for i, (act, types, shape) in enumerate([("sigmoid", (F32, F32), (37, 90)), ("tanh", (B16, B16), (3, 6, 130)),
                                             ("none", (F32, B16), (21, 2051))]):
        check(inputs(shape, *types, post, pre, gate, scale, seed=17 + i), post, pre, act)


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 255, 4097, 6001])
def test_row_counts(rows):
    check(inputs((rows, 72), F32, F32, "layer", "layer", "row", "one", seed=rows), "layer", "layer", "sigmoid")
    check(inputs((rows, 1100), B16, B16, "rms", "layer", "col", "col", seed=rows), "rms", "layer", "tanh")
    check(inputs((rows, 30), B16, B16, "layer", "rms", "full", "col", seed=rows), "layer", "rms", "tanh")
    check(inputs((rows, 200), F32, B16, "rms", "layer", "row", "col", seed=rows), "rms", "layer", "sigmoid")
    check(inputs((rows, 700), F32, F32, "layer", "rms", "full", "one", seed=rows), "layer", "rms", "sigmoid")
    if rows < 1000:
        check(inputs((rows, 9001), F32, F32, "layer", "layer", "col", "one", seed=rows), "layer", "layer", "sigmoid")


@pytest.mark.parametrize("use", [(True, False), (False, True)])
def test_one_upstream_gradient(use):
    check(inputs((40, 900), F32, F32, "layer", "rms", "full", "col", seed=3), "layer", "rms", "sigmoid", use_dr=use[0],
          use_dy=use[1])
    check(inputs((40, 1500), B16, B16, "rms", "layer", "row", "one", seed=4), "rms", "layer", "tanh", use_dr=use[0],
          use_dy=use[1])


@pytest.mark.parametrize("types", [(F32, F32), (B16, B16)])
def test_entry_norm(types):
    t = inputs((33, 901), *types, None, "layer", None, None, seed=5, with_h=False)
    check(t, None, "layer", "sigmoid", use_dr=False)


def test_entry_norm_into_bf16():
    from scpair_amd import ops
    t = inputs((33, 900), F32, F32, None, "rms", None, None, seed=6, with_h=False)
    x = t["x"].cuda().requires_grad_()
    r, y = ops.gated_residual_norm(x, pre="rms", pre_weight=t["pre_weight"].cuda(), out_dtype=B16)
    assert r is x and y.dtype == B16
    ref = {n: None if t[n] is None else t[n].double() for n in NAMES}
    close("y", y, oracle(ref, None, "rms", "none", 1e-5)[1], 33, False, B16)
    y.sum().backward()
    assert x.grad.shape == x.shape


def test_strides_and_alignment():
    """Rows inside a wider tensor, starting at any element; columns that are not next to each other are copied."""
    def padded(v):
        if v.ndim != 2:
            return v
        wide = torch.full((v.shape[0], v.shape[1] + 5), float("nan"), dtype=v.dtype, device=v.device)
        wide[:, 3:3 + v.shape[1]] = v
        return wide[:, 3:3 + v.shape[1]].detach()

    def transposed(v):
        return v.t().contiguous().t().detach() if v.ndim == 2 else v

    for layout in (padded, transposed):
        for types in TYPES:
            check(inputs((19, 333), *types, "layer", "rms", "full", "col", seed=8), "layer", "rms", "sigmoid", layout=layout)
            check(inputs((19, 1601), *types, "rms", "layer", "full", "one", seed=9), "rms", "layer", "tanh", layout=layout)


def test_broadcast_rows():
    """A stride of zero: the same block output for every row; its gradient is summed by autograd."""
    from scpair_amd import ops
    g = torch.Generator().manual_seed(1)
    x, h = torch.randn(50, 200, generator=g), torch.randn(1, 200, generator=g)
    up = torch.randn(50, 200, generator=g)
    hr = h.double().requires_grad_()
    want, = torch.autograd.grad(oracle(dict.fromkeys(NAMES) | {"x": x.double(), "h": hr.expand(50, 200)}, "layer", "rms",
                                       "none", 1e-5)[1], hr, up.double())
    hg = h.cuda().requires_grad_()
    got, = torch.autograd.grad(ops.gated_residual_norm(x.cuda(), hg.expand(50, 200), post="layer", pre="rms")[1], hg, up.cuda())
    close("dh", got, want, 50, True, F32)


def test_far_from_zero():
    """Rows whose mean is 1000 times their spread: the variance is taken about the mean.  x itself carries its mean with a
    relative error of 2^-24, i.e. 1000 * 2^-24 of the spread, in each of the few operations of the centred values."""
    from scpair_amd import ops
    g = torch.Generator().manual_seed(2)
    x = (1000 + torch.randn(16, 1500, generator=g)).float()
    y = ops.gated_residual_norm(x.cuda(), pre="layer")[1].double().cpu()
    want = _norm(x.double(), "layer", None, None, 1e-5)
    assert (y - want).abs().max().item() <= 8 * 1000 * 2.0 ** -24 * 4


def test_extremes_stay_in_their_row():
    """A row of zeros, equal values, a NaN and an infinity: other rows' outputs and gradients do not change by a bit; a row
    without spread has finite outputs and gradients."""
    from scpair_amd import ops
    for D in (900, 3000):
        g = torch.Generator().manual_seed(D)
        x, h, gate = (torch.randn(12, D, generator=g).cuda() for _ in range(3))
        up = torch.randn(12, D, generator=g).cuda()

        def run(x, h):
            x, h, gt = x.clone().requires_grad_(), h.clone().requires_grad_(), gate.clone().requires_grad_()
            r, y = ops.gated_residual_norm(x, h, gate=gt, post="layer", pre="layer", scale=0.7)
            return [r.detach(), y.detach(), *torch.autograd.grad((r, y), (x, h, gt), (up, up))]

        base = run(x, h)
        x2, h2 = x.clone(), h.clone()
        x2[0], h2[0] = 0.0, 0.0
        x2[1], h2[1] = 2.0, -3.0
        h2[2, 5] = float("nan")
        x2[3, D - 1] = float("inf")
        other = run(x2, h2)
        for a, b in zip(base, other):
            assert torch.equal(a[4:], b[4:])
            assert torch.isfinite(b[:2]).all()


def test_reproducible_and_on_another_stream():
    from scpair_amd import ops
    t = inputs((3000, 700), B16, B16, "layer", "rms", "full", "col", seed=12)
    first = check(t, "layer", "rms", "sigmoid")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = check(t, "layer", "rms", "sigmoid")
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip([*first[:2], *first[2]], [*second[:2], *second[2]]):
        assert torch.equal(a, b)


def test_frozen_parameters_and_no_grad():
    from scpair_amd import ops
    t = {n: None if v is None else v.cuda() for n, v in inputs((64, 300), F32, F32, "layer", "layer", "full", "col", 13).items()}
    kw = kwargs(t, "layer", "layer", "sigmoid", 1e-5)
    with torch.no_grad():
        r0, y0 = ops.gated_residual_norm(t["x"], t["h"], **kw)
    h = t["h"].clone().requires_grad_()
    r, y = ops.gated_residual_norm(t["x"], h, **kw)
    assert torch.equal(r, r0) and torch.equal(y, y0) and not y0.requires_grad
    dh, = torch.autograd.grad((r, y), h, (t["dr"], t["dy"]))
    full = {n: None if t[n] is None else t[n].clone().requires_grad_() for n in NAMES}
    r, y = ops.gated_residual_norm(full["x"], full["h"], **kwargs(full, "layer", "layer", "sigmoid", 1e-5))
    assert torch.equal(dh, torch.autograd.grad((r, y), full["h"], (t["dr"], t["dy"]))[0])


def test_gradient_against_differences():
    """Central differences of a scalar of the fp32 forward, step 2^-7: truncation ~ step^2 = 6e-5 of a third derivative of
    order 1, rounding ~ 64 * 2^-24 * |loss terms| / step; 2e-2 relative to the gradient's norm covers both."""
    from scpair_amd import ops
    t = {n: None if v is None else v.cuda() for n, v in inputs((6, 40), F32, F32, "layer", "layer", "full", "col", 21).items()}

    def loss(v):
        r, y = ops.gated_residual_norm(v["x"], v["h"], **kwargs(v, "layer", "layer", "tanh", 1e-5))
        return (r.double() * t["dr"].double()).sum() + (y.double() * t["dy"].double()).sum()

    leaves = {n: t[n].clone().requires_grad_() for n in NAMES}
    loss(leaves).backward()
    g = torch.Generator().manual_seed(3)
    for n in NAMES:
        d = torch.randn(t[n].shape, generator=g).cuda()
        up, dn = dict(t), dict(t)
        up[n], dn[n] = t[n] + d / 128, t[n] - d / 128
        with torch.no_grad():
            num = (loss(up) - loss(dn)).item() * 64
        ana = (leaves[n].grad.double() * d.double()).sum().item()
        assert abs(num - ana) <= 2e-2 * (leaves[n].grad.norm().item() * d.norm().item()), (n, num, ana)


def test_captured_and_replayed():
    """Forward and backward captured into one graph; replayed on new values with eager work between the replays."""
    from scpair_amd import ops
    ts = [inputs((50, 1200), B16, B16, "rms", "layer", "full", "one", seed=s) for s in (1, 2, 3)]
    names = [n for n in NAMES if ts[0][n] is not None]

    def step(v):
        r, y = ops.gated_residual_norm(v["x"], v["h"], **kwargs(v, "rms", "layer", "sigmoid", 1e-5))
        return [r, y, *torch.autograd.grad((r, y), [v[n] for n in names], (v["dr"], v["dy"]))]

    def leaves(t):
        return {n: None if t[n] is None else t[n].cuda().requires_grad_(n in names) for n in (*NAMES, "dr", "dy")}

    held = leaves(ts[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held)
    for t in ts:
        with torch.no_grad():
            for n in (*names, "dr", "dy"):
                held[n].copy_(t[n])
        graph.replay()
        torch.cuda.synchronize()
        got = [o.detach().clone() for o in outs]
        for a, b in zip(got, step(leaves(t))):
            assert torch.equal(a, b)


def test_empty_batch():
    from scpair_amd import ops
    x, h = torch.empty(0, 64, device="cuda", requires_grad=True), torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    r, y = ops.gated_residual_norm(x, h, post="layer", post_weight=w, pre="rms", pre_weight=w)
    assert r.shape == y.shape == (0, 64)
    (r.sum() + y.sum()).backward()
    assert x.grad.shape == (0, 64) and not w.grad.any()


def test_offsets_beyond_32_bits():
    """5.4 GB of rows: the last ones are computed like a small call's."""
    from scpair_amd import ops
    rows, D = 330_000, 8192
    x = torch.zeros(rows, D, dtype=B16, device="cuda")
    h = torch.zeros(rows, D, dtype=B16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    x[-4:] = torch.randn(4, D, generator=g, device="cuda").to(B16)
    h[-4:] = torch.randn(4, D, generator=g, device="cuda").to(B16)
    with torch.no_grad():
        r, y = ops.gated_residual_norm(x, h, post="rms", pre="layer")
        r4, y4 = ops.gated_residual_norm(x[-4:].clone(), h[-4:].clone(), post="rms", pre="layer")
    assert torch.equal(r[-4:], r4) and torch.equal(y[-4:], y4) and not r[:-4].any()


def test_second_derivative_is_refused():
    from scpair_amd import ops
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    _, y = ops.gated_residual_norm(x)
    g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
