"""The residual-trunk operators in calls that their documentation allows, at the ends of their ranges and in other hands: the longest
sides, more than 2^31 elements, two host threads, torch's graphed callables."""
import math
import threading

import pytest
import torch

import scpair_amd as S
from scpair_amd import ops
from tests.test_ckpt8_gpu import B16, E, F32, bound, half_step, pack_ref

pytestmark = pytest.mark.gpu


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("M,K,N", [(171, 3, 1 << 20), (5, 1 << 20, 3), (171, 8, (1 << 20) - 3), (3, (1 << 20) - 1, 9)])
@pytest.mark.parametrize("dtype", [F32, B16])
def test_linear8_longest_sides(M, K, N, dtype):
    """2^20 inputs or outputs: rows of a prepared fp32 operand are 6 * 2^20 elements long."""
    x, W = rnd(1, M, K).to(dtype).requires_grad_(), (rnd(2, N, K) / math.sqrt(K)).to(dtype).requires_grad_()
    b, up = rnd(3, N).requires_grad_(), rnd(4, M, N).to(dtype)
    y = ops.linear8(x, W, b)
    dx, dW, db = torch.autograd.grad(y, (x, W, b), up)
    xd, Wd, ud = (t.detach().cpu().double() for t in (x, W, up))
    v = pack_ref(x.detach().cpu())[2]
    m, split = (1, 0.0) if dtype == B16 else (6, 2.0 ** -22)
    cols = torch.unique(torch.cat([torch.arange(0, N, max(N // 50, 1)), torch.arange(max(N - 70, 0), N)]))      # of y and of dW's rows

    def near(got, left, right, k, add=0.0):
        want = left @ right + add
        err = bound(left, right, k) + split * (left.abs() @ right.abs()) + 4 * E + (half_step(want, B16) if dtype == B16 else E * want.abs())
        return ((got.detach().cpu().double() - want).abs() <= err).all()

    assert near(y[:, cols.cuda()], xd, Wd[cols].t(), m * K, b.detach().cpu().double()[cols])
    assert near(dx, ud, Wd, m * N)
    assert near(dW[cols.cuda()], ud.t()[cols], v, m // 2 * M if m == 6 else M)
    assert ((db.cpu().double() - ud.sum(0)).abs() <= (M / 16 + 16) * E * ud.abs().sum(0)).all()


def test_more_than_2_31_elements():
    """What is at the end of a long tensor comes out as it does alone."""
    x = torch.zeros(600_000, 5003, dtype=B16, device="cuda")
    x[-3:] = rnd(5, 3, 5003).to(B16)
    x.requires_grad_()
    a = ops.act8(x, "gelu")
    up = torch.ones_like(a)
    d, = torch.autograd.grad(a, x, up)
    tail = x.detach()[-3:].clone().requires_grad_()
    b = ops.act8(tail, "gelu")
    assert torch.equal(a[-3:], b) and torch.equal(d[-3:], torch.autograd.grad(b, tail, up[-3:])[0])
    assert not a.detach()[:-3].any() and (d[:-3] == 0.5).all()
    del a, d, up
    p, q = ops.pack8(x.detach()), ops.pack8(tail.detach())
    assert torch.equal(p.codes[-3:], q.codes) and torch.equal(p.steps[-3:], q.steps) and not p.codes[:-3].any()
    out = ops.unpack8(p)
    assert torch.equal(out[-3:], ops.unpack8(q)) and not out[:-3].any()
    del out, p
    W = rnd(6, 2, 5003).to(B16)
    with torch.no_grad():
        y = ops.linear8(x, W)
        # (the kernel may be another one for three rows: fp32 sums in another order, one rounding)
        z = tail.detach().double() @ W.double().t()
        assert ((y[-3:].double() - z).abs() <= (bound(tail.detach().double(), W.double().t(), 5003) + half_step(z, B16))).all()
        assert not y[:-3].any()


def test_longest_rows_of_a_checkpoint():
    x = torch.zeros(2, 1 << 24, device="cuda")
    x[:, -100:] = rnd(7, 2, 100)
    p = ops.pack8(x)
    # the last 128 columns: two whole groups
    codes, steps, v = pack_ref(x[:, -128:].cpu())
    assert torch.equal(p.codes[:, -128:].cpu(), codes) and torch.equal(p.steps[:, -2:].cpu(), steps) and not p.codes[:, :-128].any()
    assert torch.equal(ops.unpack8(p)[:, -128:].cpu().double(), v)
    for call in (ops.pack8, ops.act8):
        with pytest.raises(ValueError, match="columns"):
            call(torch.zeros(1, (1 << 24) + 1, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, B16])
def test_gradient_of_the_bias_alone(dtype):
    for M, N in ((1, 1), (5, 3), (300, 900), (4100, 2000)):
        b, up = torch.zeros(N, device="cuda", requires_grad=True), rnd(M, M, N).to(dtype)
        db, = torch.autograd.grad(ops.linear8(rnd(8, M, 40).to(dtype), rnd(9, N, 40).to(dtype), b), b, up)
        u = up.cpu().double()
        assert ((db.cpu().double() - u.sum(0)).abs() <= (M / 16 + 16) * E * u.abs().sum(0)).all()


def step(net, x, up):
    x = x.clone().requires_grad_()
    return [t.clone() for t in torch.autograd.grad(net(x), [x, *net.parameters()], up)]


def test_two_threads_with_streams_of_their_own():
    """Two networks trained from two host threads, each on its own stream, give what they give one after the other."""
    torch.manual_seed(0)
    nets = [S.ResidualTrunk(136, 2, gate="sigmoid", block_dtype=t).cuda() for t in (F32, B16)]
    data = [(rnd(11 + i, 200, 136), rnd(21 + i, 200, 136).to(t)) for i, t in enumerate((F32, B16))]
    want = [step(n, *d) for n, d in zip(nets, data)]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = step(nets[i], *data[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # noqa: BLE001 (shown by the assertion below)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", [F32, B16])
def test_graphed_callable(dtype):
    """torch.cuda.make_graphed_callables of a trunk: forward and backward as two graphs, replayed with eager work in between."""
    torch.manual_seed(1)
    net = S.ResidualTrunk(200, 2, norm="rms", block_dtype=dtype).cuda()
    eager = S.ResidualTrunk(200, 2, norm="rms", block_dtype=dtype).cuda()
    eager.load_state_dict(net.state_dict())
    graphed = torch.cuda.make_graphed_callables(net, (rnd(31, 64, 200).requires_grad_(),))
    for i in range(4):
        x, up = rnd(40 + i, 64, 200), rnd(50 + i, 64, 200).to(dtype)
        runs = []
        for f, params in ((graphed, net), (eager, eager)):
            xl = x.clone().requires_grad_()
            params.zero_grad(set_to_none=True)
            y = f(xl)
            y.backward(up)
            torch.cuda.synchronize()
            runs.append([y.detach().clone(), xl.grad.clone(), *(p.grad.clone() for p in params.parameters())])
        assert all(torch.equal(a, b) for a, b in zip(*runs)), i
