"""8-bit activation checkpoints (csrc/ckpt8.hip, the q8 form of csrc/wgemm.hip) against their definition in 64 bits on the
CPU.

Tolerances.  Packing is exact by its definition (power-of-two steps), so codes, steps and unpacked values are compared bit
for bit.  Activations: one fp32 evaluation of some 20 operations on values of order |z|, 32 * 2^-24 * max(|z|, 1) * |dout|, and half a step of
the output's type.  Products of K bf16 terms are exact in fp32, their sum in fp32 is off by at most sqrt-free bound
K * 2^-24 * sum|terms| in the worst order; the blocked order of the kernels (64-deep tiles into one accumulator) keeps it
below (K / 16 + 16) * 2^-24 * sum |a b|, which is computed from the operands' absolute values; the fp32 mode's operand
split leaves 2^-22 per product on top and makes the sum six times as long (dW: three times).  Outputs held in bf16: half a step, 2^-8 relative."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, B16 = torch.float32, torch.bfloat16
E = 2.0 ** -24


def pack_ref(x):
    """codes, steps (as the kernels store them) and values in float64 of a 2-D CPU tensor"""
    rows, cols = x.shape
    ld = (cols + 63) // 64 * 64
    t = torch.zeros(rows, ld, dtype=torch.float64)
    t[:, :cols] = x.double()
    t = t.reshape(rows, ld // 64, 64)
    bad = ~torch.isfinite(t).all(2)
    top = torch.where(torch.isfinite(t), t.abs(), 0.0).amax(2)
    k = torch.full_like(top, -126, dtype=torch.int64)
    for p in range(-126, 121):                       # the smallest k <= 121 with top <= 127 * 2^k
        k = torch.where(top > 127.0 * 2.0 ** p, p + 1, k)
    step = ((k + 1023) << 52).view(torch.float64)
    c = torch.round(t / step[..., None]).clamp(-127, 127)
    c = torch.where(bad[..., None], 0.0, c)
    v = torch.where(bad[..., None], float("nan"), c * step[..., None])
    return (c.reshape(rows, ld).to(torch.int8), torch.where(bad, 255, k + 127).to(torch.uint8), v.reshape(rows, ld)[:, :cols])


def rand(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    x[:, ::37] *= 20
    return x.to(dtype)


SHAPES = [(1, 1), (1, 64), (3, 7), (5, 63), (5, 65), (2, 128), (130, 200), (33, 901), (257, 1800), (4, 20001), (5000, 64)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [F32, B16])
def test_pack_and_unpack_are_exact(shape, dtype):
    from scpair_amd import ops
    x = rand(*shape, dtype, sum(shape))
    p = ops.pack8(x.cuda())
    codes, steps, v = pack_ref(x)
    assert torch.equal(p.codes.cpu(), codes) and torch.equal(p.steps.cpu(), steps)
    assert p.nbytes == codes.numel() + steps.numel() and p.shape == x.shape and p.dtype == dtype
    for t in (F32, B16):
        out = ops.unpack8(p, t)
        assert out.dtype == t and torch.equal(out.cpu().double(), v)
    assert torch.equal(ops.unpack8(p).cpu().double(), v) and ops.unpack8(p).dtype == dtype
    # packing what was unpacked changes nothing
    assert torch.equal(ops.unpack8(ops.pack8(ops.unpack8(p))).cpu().double(), v)


def test_pack_borders_of_the_step():
    """Maxima on both sides of 127 * 2^k, ties, zeros, the smallest and largest magnitudes."""
    from scpair_amd import ops
    rows = []
    for top in (127.0, math.nextafter(127.0, 200) and 127.00001, 126.99999, 128.0, 64.0, 1.0, 1.984375, 1.9843751, 3.0e38,
                3.4028234e38, 1e-38, 1.2e-38, 1e-40, 1e-45, 127 * 2.0 ** -126, 128 * 2.0 ** -126, 0.0):
        r = torch.linspace(-1, 1, 64) * 0.9
        r = (r * top).float()
        r[5], r[6] = top, -top
        rows.append(r)
    ties = torch.arange(-64, 0).float() + 0.5
    ties[0] = 127.0
    rows.append(ties)
    x = torch.stack(rows)
    codes, steps, v = pack_ref(x)
    p = ops.pack8(x.cuda())
    assert torch.equal(p.steps.cpu(), steps)
    assert torch.equal(p.codes.cpu(), codes)
    assert torch.equal(ops.unpack8(p).cpu().double(), v)


def test_non_finite_groups_read_as_nan():
    from scpair_amd import ops
    x = rand(6, 200, F32, 3)
    x[0, 3], x[1, 70], x[2, 199], x[3, 128] = float("nan"), float("inf"), -float("inf"), float("nan")
    codes, steps, v = pack_ref(x)
    p = ops.pack8(x.cuda())
    assert torch.equal(p.codes.cpu(), codes) and torch.equal(p.steps.cpu(), steps)
    out = ops.unpack8(p).cpu().double()
    assert torch.equal(out.isnan(), v.isnan()) and torch.equal(out.nan_to_num(), v.nan_to_num())


def test_pack_strides_shapes_and_empty():
    from scpair_amd import ops
    wide = rand(40, 333, B16, 4)
    for view in (wide[:, 5:205], wide[::2, 1:], wide.t(), wide[3:4].expand(7, 333), wide.reshape(8, 5, 333), wide[0]):
        dense = view.contiguous()
        got = ops.unpack8(ops.pack8(view.cuda() if view.is_contiguous() else _as_laid_out(view)))
        assert got.shape == view.shape
        want = pack_ref(dense.reshape(-1, dense.shape[-1]))[2].reshape(dense.shape)
        assert torch.equal(got.cpu().double(), want)
    for shape in ((0, 5), (5, 0), (0, 0)):
        assert ops.unpack8(ops.pack8(torch.empty(shape, device="cuda"))).shape == shape


def _as_laid_out(view):
    """the same view on the GPU (strides kept)"""
    base = view._base.cuda()
    return torch.as_strided(base, view.size(), view.stride(), view.storage_offset())


def act_ref(z, kind, slope):
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    return torch.where(z > 0, z, slope * z)


def act_slope_ref(v, kind, slope):
    if kind == "gelu":
        return torch.special.ndtr(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if kind == "silu":
        return torch.sigmoid(v) * (1 + v * torch.sigmoid(-v))
    return torch.where(v > 0, 1.0, slope)


def half_step(want, dtype):
    return want.abs() * (2.0 ** -8 if dtype == B16 else E)


@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (33, 901), (130, 1024), (2, 5, 70)])
@pytest.mark.parametrize("kind,slope", [("gelu", 0.0), ("silu", 0.0), ("leaky_relu", 0.01), ("leaky_relu", 0.0)])
@pytest.mark.parametrize("dtype", [F32, B16])
def test_act8(shape, kind, slope, dtype):
    from scpair_amd import ops
    g = torch.Generator().manual_seed(5)
    z, up = (3 * torch.randn(shape, generator=g)).to(dtype), torch.randn(shape, generator=g).to(dtype)
    zg = z.cuda().requires_grad_()
    a = ops.act8(zg, kind, slope)
    want = act_ref(z.double(), kind, slope)
    assert a.dtype == dtype and a.shape == z.shape
    assert ((a.detach().cpu().double() - want).abs() <= 32 * E * z.double().abs().clamp(min=1) + half_step(want, dtype)).all()
    dz, = torch.autograd.grad(a, zg, up.cuda())
    v = pack_ref(z.reshape(-1, shape[-1]))[2].reshape(shape)
    want = up.double() * act_slope_ref(v, kind, slope)
    assert dz.dtype == dtype
    assert ((dz.cpu().double() - want).abs() <= 32 * E * up.double().abs() * v.abs().clamp(min=1) + half_step(want, dtype)).all()
    with torch.no_grad():
        assert torch.equal(ops.act8(zg, kind, slope), a)


def test_act8_extremes():
    """Large magnitudes neither overflow nor lose their sign; an infinity gives its own limit forward and NaN backward."""
    from scpair_amd import ops
    z = torch.tensor([[-3e38, -1e4, -100.0, -20.0, 0.0, 20.0, 100.0, 1e4, 3e38]])
    for kind in ("gelu", "silu"):
        a = ops.act8(z.cuda(), kind).cpu()
        assert torch.isfinite(a).all() and (a[0, 5:] == z[0, 5:]).all() and (a[0, :4].abs() <= 1e-7).all()
    x = torch.zeros(2, 64)
    x[0, 1] = float("inf")
    xg = x.cuda().requires_grad_()
    a = ops.act8(xg, "silu")
    assert a[0, 1] == float("inf")
    d, = torch.autograd.grad(a.sum(), xg)
    assert d[0].isnan().all() and torch.isfinite(d[1]).all()


def bound(a, b, k):
    return (k / 16 + 16) * E * (a.abs() @ b.abs())


LINEARS = [(1, 1, 1), (1, 8, 5), (3, 65, 7), (64, 64, 64), (130, 901, 33), (257, 300, 517), (777, 1801, 901), (1024, 900, 1800),
           (2049, 72, 264), (5000, 130, 70), (2500, 1030, 3100)]


@pytest.mark.parametrize("M,K,N", LINEARS)
@pytest.mark.parametrize("xt,wt,mode", [(B16, B16, "fp32"), (B16, F32, "fp32"), (F32, F32, "fp32"), (F32, F32, "bf16")])
@pytest.mark.parametrize("bias", [True, False])
def test_linear8(M, K, N, xt, wt, mode, bias):
    from scpair_amd import ops
    g = torch.Generator().manual_seed(M + K + N)
    x, W = rand(M, K, xt, M), (torch.randn(N, K, generator=g) / math.sqrt(K)).to(wt)
    x = x.clamp(-50, 50)
    b = 0.1 * torch.randn(N, generator=g) if bias else None
    up = torch.randn(M, N, generator=g).to(xt)
    old = ops.get_precision()
    ops.set_precision(mode)
    try:
        leaves = [t.cuda().requires_grad_() for t in (x, W, b) if t is not None]
        y = ops.linear8(*leaves)
        grads = torch.autograd.grad(y, leaves, up.cuda())
        again = torch.autograd.grad(ops.linear8(*leaves), leaves, up.cuda())
        with torch.no_grad():
            assert torch.equal(ops.linear8(*leaves), y)
    finally:
        ops.set_precision(old)
    for a, c in zip(grads, again):
        assert torch.equal(a, c)
    narrow = xt == B16 or mode == "bf16"                  # products of bf16 operands
    r = (lambda t: t.to(B16).double()) if narrow else (lambda t: t.double())
    v = pack_ref(x)[2]
    split = 0.0 if narrow else 2.0 ** -22
    xr, Wr, ur = r(x), r(W), r(up)

    def close(name, got, want, err, dtype):
        assert got.dtype == dtype and got.shape == want.shape, name
        over = (got.detach().cpu().double() - want).abs() - err - (half_step(want, dtype) if dtype == B16 else E * want.abs())
        assert over.max().item() <= 0, f"{name}: {(got.detach().cpu().double() - want).abs().max().item()}"

    want = xr @ Wr.t() + (b.double() if bias else 0)
    close("y", y, want, bound(xr, Wr.t(), K if narrow else 6 * K) + split * (xr.abs() @ Wr.t().abs()) + 4 * E, xt)
    close("dx", grads[0], ur @ Wr, bound(ur, Wr, N if narrow else 6 * N) + split * (ur.abs() @ Wr.abs()), xt)
    close("dW", grads[1], ur.t() @ v, bound(ur.t(), v, M if narrow else 3 * M) + split * (ur.t().abs() @ v.abs()), wt)
    if bias:
        close("db", grads[2], up.double().sum(0), (M / 16 + 16) * E * up.double().abs().sum(0), F32)


def test_linear8_layouts_and_partial_gradients():
    from scpair_amd import ops
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(60, 150, generator=g).to(B16).cuda()
    W = torch.randn(40, 96, generator=g).to(B16).cuda()
    base = ops.linear8(wide[:, 7:103].contiguous(), W)
    assert torch.equal(ops.linear8(wide[:, 7:103], W), base)
    assert torch.equal(ops.linear8(wide[:, 7:103].reshape(3, 20, 96), W).reshape(60, 40), base)
    assert torch.equal(ops.linear8(wide[:, 7:103], W.t().contiguous().t()), base)
    assert torch.equal(ops.linear8(wide[:, 7:103].t().contiguous().t(), W), base)
    x = wide[:, 7:103].clone().requires_grad_()
    Wl, b = W.clone().requires_grad_(), torch.zeros(40, dtype=B16, device="cuda", requires_grad=True)
    y = ops.linear8(x, Wl, b)
    dx, dW, db = torch.autograd.grad(y.float().sum(), (x, Wl, b))
    assert db.dtype == B16 and torch.equal(db.cpu(), torch.full((40,), 60.0, dtype=B16))
    xs = wide[:, 7:103].clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.linear8(xs, W).float().sum(), xs)[0], dx)
    assert torch.equal(torch.autograd.grad(ops.linear8(wide[:, 7:103], Wl).float().sum(), Wl)[0], dW)


def test_linear8_keeps_one_byte_per_element():
    from scpair_amd import ops
    W = torch.zeros(64, 4096, dtype=B16, device="cuda", requires_grad=True)
    x = torch.zeros(4096, 4096, dtype=B16, device="cuda")
    y = ops.linear8(x, W)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    del x
    assert before - torch.cuda.memory_allocated() == 4096 * 4096 * 2       # the input is free to go
    kept = torch.cuda.memory_allocated()
    del y
    assert kept - torch.cuda.memory_allocated() <= 4096 * 4096 * (1 + 1 / 64) + 4096 * 64 * 2 + 4096


def test_linear8_empty_batch_and_non_finite():
    from scpair_amd import ops
    W = torch.randn(40, 96, device="cuda").to(B16).requires_grad_()
    x = torch.empty(0, 96, dtype=B16, device="cuda", requires_grad=True)
    y = ops.linear8(x, W)
    assert y.shape == (0, 40)
    dx, dW = torch.autograd.grad(y.sum(), (x, W))
    assert dx.shape == (0, 96) and not dW.any()
    x = torch.randn(300, 200, device="cuda").to(B16)
    W = torch.randn(40, 200, device="cuda").to(B16).requires_grad_()
    x[123, 70] = float("inf")
    dW, = torch.autograd.grad(ops.linear8(x, W).float().sum(), W, retain_graph=False)
    assert dW[:, 64:128].isnan().all() and torch.isfinite(dW[:, :64]).all() and torch.isfinite(dW[:, 128:]).all()


def test_linear8_long_batch():
    """More than 2 GiB of input: forward and dx run in pieces, the weight gradient in K-ranges with their own base."""
    from scpair_amd import ops
    M, K, N = 1_100_000, 1024, 24
    x = torch.zeros(M, K, dtype=B16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for r in (0, 600_000, M - 130):
        x[r:r + 130] = torch.randn(130, K, generator=g, device="cuda").to(B16)
    W = torch.randn(N, K, generator=g, device="cuda").to(B16).requires_grad_()
    up = torch.zeros(M, N, dtype=B16, device="cuda")
    for r in (0, 600_000, M - 130):
        up[r:r + 130] = torch.randn(130, N, generator=g, device="cuda").to(B16)
    x.requires_grad_()
    y = ops.linear8(x, W)
    dx, dW = torch.autograd.grad(y, (x, W), up)
    pick = torch.cat([torch.arange(r, r + 130) for r in (0, 600_000, M - 130)]).cuda()
    xs, us = x.detach()[pick].cpu(), up[pick].cpu().double()
    Wd = W.detach().cpu().double()
    for got, want, err in ((y.detach()[pick], xs.double() @ Wd.t(), bound(xs.double(), Wd.t(), K)),
                           (dx[pick], us @ Wd, bound(us, Wd, N)),
                           (dW, us.t() @ pack_ref(xs)[2], bound(us.t(), pack_ref(xs)[2], 390))):
        got = got.cpu().double()
        assert ((got - want).abs() <= err + half_step(want, B16)).all()
    assert not y.detach()[200:600_000].any() and not dx[700_000:M - 130].any()


def test_captured_and_replayed():
    """A residual block's two Linears and its activation, forward and backward, captured once and replayed on new values."""
    from scpair_amd import ops
    g = torch.Generator(device="cuda").manual_seed(9)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(B16)
    batches = [(rn(300, 200), rn(300, 200)) for _ in range(3)]
    params = [rn(520, 200), rn(520).float(), rn(200, 520)]

    def step(x, up, W1, b1, W2):
        y = ops.linear8(ops.act8(ops.linear8(x, W1, b1), "gelu"), W2)
        return [y.detach(), *torch.autograd.grad(y, (x, W1, b1, W2), up)]

    def leaves(x, up):
        return [x.clone().requires_grad_(), up.clone(), *(p.clone().requires_grad_() for p in params)]

    held = leaves(*batches[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*held)
    for batch in batches:
        with torch.no_grad():
            for t, v in zip(held, batch):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step(*leaves(*batch))):
            assert torch.equal(a, b)


def test_relu_of_infinities():
    from scpair_amd import ops
    x = torch.tensor([[float("inf"), -float("inf"), float("nan"), -1.0, 0.0, 2.0]])
    for dtype in (F32, B16):
        a = ops.act8(x.to(dtype).cuda(), "leaky_relu", 0.0).cpu().float()
        assert a[0, 0] == float("inf") and a[0, 1] == 0 and a[0, 2].isnan() and a[0, 3:].tolist() == [0.0, 0.0, 2.0]


def _net(x, W, b):
    from scpair_amd import ops
    r, y = ops.gated_residual_norm(x, pre="rms")
    h = ops.linear8(ops.act8(ops.linear8(y, W, b), "gelu"), W.t(), None)
    return ops.gated_residual_norm(r, h, gate=y, scale=0.3, post="layer", pre="rms")[1]


@pytest.mark.parametrize("dtype", [F32, B16])
def test_backward_twice_offloaded_recomputed_and_elsewhere(dtype):
    """The same gradients, bit for bit: from a second backward pass over a kept graph, with the saved tensors moved to host
    memory in between, under activation recomputation, on another stream, and with the backward pass in the calling thread."""
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator(device="cuda").manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    x, W, b, up = rn(70, 136).requires_grad_(), rn(264, 136).requires_grad_(), rn(264).requires_grad_(), rn(70, 136)
    y = _net(x, W, b)
    first = torch.autograd.grad(y, (x, W, b), up, retain_graph=True)
    runs = [torch.autograd.grad(y, (x, W, b), up)]
    with torch.autograd.graph.save_on_cpu():
        y = _net(x, W, b)
    runs.append(torch.autograd.grad(y, (x, W, b), up))
    runs.append(torch.autograd.grad(checkpoint(_net, x, W, b, use_reentrant=False), (x, W, b), up))
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        leaves = [t.detach().clone().requires_grad_() for t in (x, W, b)]
        runs.append(torch.autograd.grad(_net(*leaves), leaves, up.clone()))
        torch.cuda.current_stream().synchronize()
    with torch.autograd.set_multithreading_enabled(False):
        runs.append(torch.autograd.grad(_net(x, W, b), (x, W, b), up))
    for run in runs:
        for a, c in zip(first, run):
            assert torch.equal(a, c)


def test_second_derivatives_are_refused():
    from scpair_amd import ops
    x = torch.randn(8, 40, device="cuda", requires_grad=True)
    W = torch.randn(16, 40, device="cuda", requires_grad=True)
    for out in (ops.act8(x, "silu"), ops.linear8(x, W)):
        d, = torch.autograd.grad(out.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            d.sum().backward()


def test_weights_changed_between_forward_and_backward_are_refused():
    from scpair_amd import ops
    x, W = torch.randn(8, 40, device="cuda", requires_grad=True), torch.randn(16, 40, device="cuda", requires_grad=True)
    y = ops.linear8(x, W)
    with torch.no_grad():
        W.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("N,K", [(1, 300), (7, 300), (300, 1), (300, 7), (9, 9)])
@pytest.mark.parametrize("xt", [F32, B16])
def test_linear8_narrow_sides_and_broadcast_rows(N, K, xt):
    """Fewer than 8 inputs or outputs, and inputs and gradients whose rows are one row (stride 0)."""
    from scpair_amd import ops
    g = torch.Generator().manual_seed(N * 1000 + K)
    x, W, up = torch.randn(1, K, generator=g).to(xt), torch.randn(N, K, generator=g).to(xt), torch.randn(1, N, generator=g).to(xt)
    M = 200
    xl, Wl = x.cuda().requires_grad_(), W.cuda().requires_grad_()
    y = ops.linear8(xl.expand(M, K), Wl)
    dxr, dW = torch.autograd.grad(y, (xl, Wl), up.cuda().expand(M, N))
    xd, Wd, ud = x.double(), W.double(), up.double()
    v = pack_ref(x)[2]
    near = lambda got, want, err: ((got.detach().cpu().double() - want).abs() <= err + half_step(want, xt) * 1.01).all()
    assert near(y, (xd @ Wd.t()).expand(M, N), bound(xd, Wd.t(), 6 * K) + 2.0 ** -20)
    assert near(dW, M * (ud.t() @ v), M * (bound(ud.t(), v, 3 * M) + 2.0 ** -20))
    # each row's dx is rounded to xt before autograd adds the rows
    assert near(dxr, M * (ud @ Wd), M * (bound(ud, Wd, 6 * N) + 2.0 ** -20 + half_step(ud @ Wd, xt) + 16 * E * (ud @ Wd).abs()))


@pytest.mark.parametrize("M,apart", [(130, 1 << 25), (3, 1 << 30)])
def test_linear8_rows_far_apart(M, apart):
    """Rows of x that no 32-bit offset reaches from one to the next give what the same rows side by side give."""
    from scpair_amd import ops
    g = torch.Generator().manual_seed(M)
    W = torch.randn(72, 64, generator=g).to(B16).cuda()
    rows = torch.randn(M, 64, generator=g).to(B16).cuda()
    far = torch.empty((M - 1) * apart + 64, dtype=B16, device="cuda").as_strided((M, 64), (apart, 1))
    far.copy_(rows)
    xd, Wd = rows.cpu().double(), W.cpu().double()
    want = xd @ Wd.t()
    with torch.no_grad():
        assert ((ops.linear8(far, W).cpu().double() - want).abs() <= bound(xd, Wd.t(), 64) + half_step(want, B16)).all()
    p, q = ops.pack8(far), ops.pack8(rows)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.steps, q.steps)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (7, 9, 200), (256, 256, 64), (300, 517, 65), (257, 255, 129), (513, 264, 4097),
                                   (1000, 777, 1000)])
def test_wide_products_at_any_size(M, N, K):
    """The three forms of the wide kernel that linear8 uses for large batches, at sizes that end inside its tiles and K-steps."""
    from scpair_amd import _lib, ops
    L = _lib.lib()
    up = lambda n: (n + 7) // 8 * 8
    g = torch.Generator().manual_seed(M + N + K)
    A, W = torch.zeros(M, up(K), dtype=B16), torch.zeros(N, up(K), dtype=B16)
    A[:, :K], W[:, :K] = torch.randn(M, K, generator=g).to(B16), torch.randn(N, K, generator=g).to(B16)
    Wc = torch.full((K, up(N)), 7.0, dtype=B16)                   # columns behind N are read, but never used
    Wc[:, :N] = W[:, :K].t()
    bias = torch.randn(N, generator=g)
    x = torch.randn(K, N, generator=g).to(B16)
    dy = torch.full((K, up(M)), 7.0, dtype=B16)
    dy[:, :M] = A[:, :K].t()
    a, w, wc, b, d = (t.cuda() for t in (A, W, Wc, bias, dy))
    p = ops.pack8(x.cuda())
    ad = A[:, :K].double()
    for c16 in (1, 0):
        ws = torch.empty(max(L.scp_gemm_bf16_ws_floats(M, N, K, N), L.scp_gemm_q8_ws_floats(M, N, K, max(up(M), p.codes.shape[1]), N), 1),
                         device="cuda")
        for col in (0, 1, 2):
            out = torch.full((M + 1, N), 3.0, dtype=B16 if c16 else F32, device="cuda")
            if col == 2:
                rc = L.scp_gemm_q8(M, N, K, d.data_ptr(), up(M), p.codes.data_ptr(), p.steps.data_ptr(), out.data_ptr(), c16, N,
                                   ws.data_ptr(), _lib.stream())
                right, add = pack_ref(x)[2], 0.0
            else:
                o = wc if col else w
                rc = L.scp_gemm_rows(col, M, N, K, a.data_ptr(), a.stride(0), o.data_ptr(), o.stride(0), out.data_ptr(), c16, N,
                                     b.data_ptr(), ws.data_ptr(), _lib.stream())
                right, add = W[:, :K].double().t(), bias.double()
            assert rc == 0
            want = ad @ right + add
            err = bound(ad, right, K) + E * want.abs() * 2 + (half_step(want, B16) * 1.01 if c16 else 0)
            assert ((out[:M].cpu().double() - want).abs() <= err).all(), (col, c16)
            assert (out[M] == 3.0).all()
