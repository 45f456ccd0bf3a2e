"""ops.gated_residual_norm where a row holds an infinity: what the formula leaves finite is finite and right, wherever in the row the
infinity stands.  Finite values that come out as exact zeros (an rms norm's 1 / spread is 0) or as plain sums and products of two
or three numbers are compared to 4 * 2^-24 relative (bf16: half a step on top)."""
import pytest
import torch

from tests.test_residual_norm_gpu import B16, F32, _norm

pytestmark = pytest.mark.gpu

# every kernel variant; positions in the first chunk, the one before the last, and the last one, which overlaps it
WIDTHS = [7, 8, 9, 30, 65, 130, 513, 900, 1025, 4099, 6145, 8193, 16383]
INF = float("inf")


def same(got, want, dtype):
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()])
    tol = want[fin].abs() * (4 * 2.0 ** -24 + (2.0 ** -8 if dtype == B16 else 0))
    assert ((got[fin] - want[fin]).abs() <= tol).all()


def places(D):
    return sorted({0, max(D - 9, 0), max(D - 8, 0), max(D - 3, 0), D - 1})


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, B16])
def test_rms_norm_of_an_infinity(D, dtype):
    from scpair_amd import ops
    at = places(D)
    g = torch.Generator().manual_seed(D)
    x = torch.randn(len(at) + 1, D, generator=g).to(dtype)
    for i, j in enumerate(at):
        x[i, j] = INF if i & 1 else -INF
    w = torch.ones(D)
    _, y = ops.gated_residual_norm(x.cuda(), pre="rms", pre_weight=w.cuda())
    want = _norm(x.double(), "rms", w.double(), None, 1e-5)
    assert (want[:-1].nan_to_num() == 0).all()
    same(y[:-1], want[:-1], dtype)
    assert torch.isfinite(y[-1]).all()
    # the same behind a block: the finite elements of r are x's
    r, _ = ops.gated_residual_norm(torch.ones_like(x).cuda(), x.cuda(), post="rms", pre="rms")
    same(r[:-1], 1 + _norm(x.double(), "rms", None, None, 1e-5)[:-1], dtype)


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, B16])
@pytest.mark.parametrize("gate", [None, "full"])
def test_infinite_gradient_without_a_post_norm(D, dtype, gate):
    """An infinity in dr stays in its element of dx and dh where no norm lies behind the block, and in its column of ds."""
    from scpair_amd import ops
    at = places(D)
    g = torch.Generator().manual_seed(D)
    rn = lambda *s: torch.randn(*s, generator=g)
    x, h, dr = (rn(len(at), D).to(dtype) for _ in range(3))
    s = 0.5 + 0.1 * rn(D).abs()
    q = (1 + rn(len(at), D).abs()).to(dtype) if gate else None
    for i, j in enumerate(at):
        dr[i, j] = INF
    leaves = [t.cuda().requires_grad_() for t in ((x, h, s) if q is None else (x, h, s, q))]
    r, _ = ops.gated_residual_norm(*leaves[:2], scale=leaves[2], gate=None if q is None else leaves[3], gate_act="none", pre="rms")
    got = torch.autograd.grad(r, leaves, dr.cuda())
    d, f = dr.double(), 1.0 if q is None else q.double()
    same(got[0], d, dtype)
    same(got[1], d * s.double() * f, dtype)
    want = (d * h.double() * f).sum(0)
    assert torch.equal(torch.isfinite(got[2]).cpu(), torch.isfinite(want)) and torch.equal(got[2].isnan().cpu(), want.isnan())
    if q is not None:
        same(got[3], d * s.double() * h.double(), dtype)


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("pre", ["rms", "layer"])
def test_gradient_of_the_stream_alone(D, pre):
    """Only r is used: dx is dr whatever the norm of the row would have been, and the norm's parameters get nothing."""
    from scpair_amd import ops
    at = places(D)
    g = torch.Generator().manual_seed(D)
    x, h, dr = (torch.randn(len(at), D, generator=g) for _ in range(3))
    for i, j in enumerate(at):
        x[i, j] = INF
    x, h, w = x.cuda().requires_grad_(), h.cuda().requires_grad_(), torch.ones(D, device="cuda", requires_grad=True)
    r, _ = ops.gated_residual_norm(x, h, pre=pre, pre_weight=w)
    dx, dh, dw = torch.autograd.grad(r, (x, h, w), dr.cuda(), allow_unused=True)
    assert torch.equal(dx.cpu(), dr) and torch.equal(dh.cpu(), dr)
    assert dw is None or not dw.any()
