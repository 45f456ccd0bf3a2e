"""ops.linear8 on each of its matrix kernels: 64 x 64 tiles straight from the tensors, 128 x 128 and 256 x 256 tiles on prepared
operands.  The kernel is chosen by a cost model of the shape; every case here asserts the choice it is meant for, so that a retuned
model cannot empty the coverage.  Values against the definition in 64 bits; tolerances are those of test_ckpt8_gpu.py."""
import ctypes as C
import math

import pytest
import torch

from scpair_amd import _lib
from tests.test_ckpt8_gpu import B16, E, F32, bound, half_step, pack_ref, rand

pytestmark = pytest.mark.gpu

# x, W, precision mode
TYPES = {"bf16": (B16, B16, "fp32"), "bf16 x, fp32 W": (B16, F32, "fp32"), "fp32 in bf16 mode": (F32, F32, "bf16"), "fp32": (F32, F32, "fp32")}


def tiles_of(M, K, N, kind):
    """tile edges of y, dx and dW for contiguous tensors"""
    xt, wt, mode = TYPES[kind]
    a = _lib.Linear8()
    for k, v in dict(x=4096, W=4096, dy=4096, M=M, N=N, K=K, ldx=K, lddy=N, x_bf16=xt == B16, w_bf16=wt == B16,
                     ns=3 if xt == F32 and mode == "fp32" else 1).items():
        setattr(a, k, v)
    t = (C.c_int * 3)()
    assert _lib.lib().scp_linear8_tiles(C.byref(a), t) == 0
    return tuple(t)


@pytest.mark.parametrize("kind,M,K,N,tile", [("bf16", 64, 128, 64, 64), ("fp32", 65, 130, 67, 64), ("bf16", 8, 2184, 2312, 128),
                                             ("fp32", 2952, 2200, 8, 128), ("bf16", 8, 2838, 2883, 256)])
def test_weight_gradient_of_the_largest_inputs(kind, M, K, N, tile):
    """Groups of the largest step, 2^121: max|x| above 127 * 2^120 = 1.69e38, here 3e38 beside zeros and values that round to 0
    and 1.  dW is finite for the upstream gradients of 1e-3 in those rows, and for 0, the lowest value of the type among them."""
    from scpair_amd import ops
    xt, wt, mode = TYPES[kind]
    assert tiles_of(M, K, N, kind)[2] == tile
    g = torch.Generator().manual_seed(M)
    x, W = torch.randn(M, K, generator=g).to(xt), (0.01 * torch.randn(N, K, generator=g)).to(wt)
    up = torch.randn(M, N, generator=g).to(xt)
    x[1, 70], x[1, 71], x[1, 72], x[1, 73] = 3e38, -1.8e38, 3e36, 0.0
    x[5, 3] = torch.finfo(xt).min
    x[6, K - 1] = 1.7e38
    up[1], up[5], up[6] = 1e-3, 0.0, 1e-3
    Wl = W.cuda().requires_grad_()
    dW, = torch.autograd.grad(ops.linear8(x.cuda(), Wl), Wl, up.cuda())
    v, ud = pack_ref(x)[2], up.double()
    want = ud.t() @ v
    err = bound(ud.t(), v, M if xt == B16 else 3 * M) + (0 if xt == B16 else 2.0 ** -22 * (ud.t().abs() @ v.abs()))
    over = (dW.cpu().double() - want).abs() - err - (half_step(want, B16) if wt == B16 else E * want.abs())
    assert torch.isfinite(dW).all() and over.max().item() <= 0


# smallest shapes that each kernel takes, aligned and ragged, alone and together
CASES = [
    ("bf16", 2254, 8, 2284, (128, 64, 64)), ("bf16", 2285, 1227, 3172, (128, 64, 64)), ("bf16 x, fp32 W", 3057, 1968, 2390, (128, 64, 256)),
    ("bf16 x, fp32 W", 6184, 992, 1224, (128, 128, 256)), ("fp32", 8, 841, 9, (128, 64, 64)), ("fp32", 24, 912, 8, (128, 64, 64)),
    ("bf16", 4116, 8, 1975, (256, 64, 64)), ("bf16", 4674, 69, 5660, (256, 64, 64)), ("fp32 in bf16 mode", 3004, 247, 5184, (256, 64, 64)),
    ("fp32", 2374, 10, 4264, (256, 64, 64)), ("fp32", 1773, 1435, 1764, (256, 64, 64)),
    ("fp32", 10, 12, 789, (64, 128, 64)), ("bf16", 5536, 912, 8, (64, 128, 64)), ("bf16", 3380, 2161, 833, (64, 128, 128)),
    ("fp32 in bf16 mode", 4964, 1489, 870, (64, 128, 256)), ("fp32", 2884, 2493, 8, (64, 128, 128)), ("fp32", 2563, 2107, 609, (64, 64, 128)),
    ("bf16", 1837, 5384, 9, (64, 256, 64)), ("fp32", 1950, 4356, 9, (64, 256, 128)), ("bf16", 5015, 5321, 76, (64, 256, 128)),
    ("bf16", 8, 2849, 1846, (64, 64, 128)), ("fp32 in bf16 mode", 9, 1784, 4677, (64, 64, 256)), ("bf16", 8, 2064, 4056, (64, 64, 256)),
    ("bf16", 3000, 1500, 4000, (256, 256, 256)), ("bf16", 3001, 1501, 4003, (256, 256, 256)),
    ("bf16 x, fp32 W", 3001, 1501, 4003, (256, 256, 256)), ("fp32 in bf16 mode", 3000, 1504, 4003, (256, 256, 256)),
    ("fp32", 1745, 2913, 5343, (256, 256, 256)),
]


def some(n, seed):
    """up to 200 rows: the first and last ones, those at the borders of tiles, and a few others"""
    pick = {0, 1, n - 1, n - 2, *(b + d for b in range(64, n, 256) for d in (-1, 0)), *(b + d for b in range(256, n, 512) for d in (-1, 0)),
            *torch.randint(0, n, (40,), generator=torch.Generator().manual_seed(seed)).tolist()}
    return torch.tensor(sorted(i for i in pick if 0 <= i < n)[:200])


@pytest.mark.parametrize("kind,M,K,N,tiles", CASES)
@pytest.mark.parametrize("strided", [False, True])
def test_every_kernel(kind, M, K, N, tiles, strided):
    """Outputs, gradients and the checkpoint that is kept.  strided: x and dy are column ranges of wider tensors at odd offsets (the
    choice may then be another one, the values may not)."""
    from scpair_amd import ops
    xt, wt, mode = TYPES[kind]
    if not strided:
        assert tiles_of(M, K, N, kind) == tiles
    g = torch.Generator().manual_seed(M + K + N)
    x = rand(M, K, xt, M).clamp(-50, 50)
    W, b = (torch.randn(N, K, generator=g) / math.sqrt(K)).to(wt), 0.1 * torch.randn(N, generator=g)
    up = torch.randn(M, N, generator=g).to(xt)
    lay = lambda t: torch.cat([t[:, :3], t, t[:, :2]], 1).cuda()[:, 3:-2] if strided else t.cuda()
    old = ops.get_precision()
    ops.set_precision(mode)
    kept = []
    try:
        leaves = [lay(x).detach().requires_grad_(), W.cuda().requires_grad_(), b.cuda().requires_grad_()]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
            y = ops.linear8(*leaves)
        dx, dW, db = torch.autograd.grad(y, leaves, lay(up))
        again = torch.autograd.grad(ops.linear8(*leaves), leaves, lay(up))
    finally:
        ops.set_precision(old)
    assert all(torch.equal(p, q) for p, q in zip((dx, dW, db), again))
    codes, steps, v = pack_ref(x)
    assert any(t.dtype == torch.int8 and torch.equal(t.cpu(), codes) for t in kept)
    assert any(t.dtype == torch.uint8 and torch.equal(t.cpu(), steps) for t in kept)
    narrow = kind != "fp32"
    r = (lambda t: t.to(B16).double()) if narrow else (lambda t: t.double())
    split = 0.0 if narrow else 2.0 ** -22
    xr, Wr, ur = r(x), r(W), r(up)
    rows, outs = some(M, 1), some(N, 2)

    def close(name, got, left, right, terms, dtype, add=0.0):
        want = left @ right + add
        err = bound(left, right, terms) + split * (left.abs() @ right.abs()) + 4 * E + (half_step(want, B16) if dtype == B16 else E * want.abs())
        assert got.dtype == dtype
        over = (got.detach().cpu().double() - want).abs() - err
        assert over.max().item() <= 0, (name, over.max().item())

    close("y", y[rows.cuda()], xr[rows], Wr.t(), K if narrow else 6 * K, xt, b.double())
    close("dx", dx[rows.cuda()], ur[rows], Wr, N if narrow else 6 * N, xt)
    close("dW", dW[outs.cuda()], ur.t()[outs], v, M if narrow else 3 * M, wt)
    want = up.double().sum(0)
    assert ((db.cpu().double() - want).abs() <= (M / 16 + 16) * E * up.double().abs().sum(0)).all()


# rows of an operand that the wide kernel addresses at once: 2 GiB less 64 KB
PIECE = ((1 << 31) - 65536) // 2


@pytest.mark.parametrize("kind,M,K,N", [("bf16", 300_001, 4096, 4096), ("bf16", 270_003, 4097, 4111), ("fp32", 45_001, 4096, 4096)])
def test_batches_beyond_2_gib(kind, M, K, N):
    """The wide kernel on operands beyond 2 GiB: y and dx in pieces, dW in K-ranges with their own base.  Rows are zero but for a few at
    both ends and on both sides of every piece's border."""
    from scpair_amd import ops
    xt, wt, _ = TYPES[kind]
    assert tiles_of(M, K, N, kind) == (256, 256, 256)
    terms = 6 if kind == "fp32" else 1
    up8 = lambda n: (n + 7) // 8 * 8
    assert terms * up8(K) * M > PIECE and terms * up8(N) * M > PIECE
    at = {0, M - 60}
    for n in (K, N):
        at |= {p for p in range(0, M, PIECE // (terms * up8(n))) if p}
    pick = torch.tensor(sorted({r for p in at for r in range(max(p - 60, 0), min(p + 60, M))})).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    W = (rn(N, K) / math.sqrt(K)).to(wt).requires_grad_()
    x, up = torch.zeros(M, K, dtype=xt, device="cuda"), torch.zeros(M, N, dtype=xt, device="cuda")
    x[pick], up[pick] = rn(len(pick), K).to(xt), rn(len(pick), N).to(xt)
    x.requires_grad_()
    y = ops.linear8(x, W)
    dx, dW = torch.autograd.grad(y, (x, W), up)
    xs, us, Wd = x.detach()[pick].cpu(), up[pick].cpu().double(), W.detach().cpu().double()
    v, outs = pack_ref(xs)[2], some(N, 3)
    split = 2.0 ** -22 if kind == "fp32" else 0.0
    for got, left, right, k in ((y.detach()[pick], xs.double(), Wd.t(), terms * K), (dx[pick], us, Wd, terms * N),
                                (dW[outs.cuda()], us.t()[outs], v, (3 if terms == 6 else 1) * len(pick))):
        want = left @ right
        err = bound(left, right, k) + split * (left.abs() @ right.abs()) + (half_step(want, B16) if got.dtype == B16 else E * want.abs())
        assert ((got.cpu().double() - want).abs() <= err).all()
    rest = torch.ones(M, dtype=torch.bool, device="cuda")
    rest[pick] = False
    assert not (y.detach().any(1) & rest).any() and not (dx.any(1) & rest).any()
