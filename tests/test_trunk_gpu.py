"""The residual-trunk operators run together as they are used (ResidualTrunk): forward and all gradients against the same
network in 64 bits on the CPU, whose Linear layers and activations take their backward pass from the same 8-bit checkpoints.

Tolerances, relative to the largest value of an output or gradient.  Outputs of fp32 blocks: three blocks of some 30 chained
operations at 2^-24 each, far below 2e-4.  Gradients of fp32 blocks: a checkpoint's code is another one where the fp32 and the
64-bit activation round to different sides of a border, about 1e-6 / 0.03 of the elements (fp32 error over step), i.e. a few
of the 10^5 here.  One such code moves one dz by |da| max|f''| step <= 4 * 0.8 * 2^-4 = 0.2 (activations up to 4, hence steps up
to 2^-4; upstream gradients up to 4), and through a weight of at most 0.1 (1 / sqrt(96) uniform) one row's gradient by 0.02 of
a largest value of 5: 4e-3.  bf16 blocks: every operator's output is rounded to 2^-8 relative, some ten roundings in a row per
block (errors add in quadrature): 6e-2.
"""
import pytest
import torch

import scpair_amd as S
from tests.test_ckpt8_gpu import act_ref, act_slope_ref, pack_ref
from tests.test_residual_norm_gpu import _norm

pytestmark = pytest.mark.gpu


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W, b):
        ctx.save_for_backward(pack_ref(x.float())[2], W)
        return x @ W.t() + b

    @staticmethod
    def backward(ctx, d):
        v, W = ctx.saved_tensors
        return d @ W, d.t() @ v, d.sum(0)


class _Act(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, kind):
        ctx.kind = kind
        ctx.save_for_backward(pack_ref(z.float())[2])
        return act_ref(z, kind, 0.01)

    @staticmethod
    def backward(ctx, d):
        v, = ctx.saved_tensors
        return d * act_slope_ref(v, ctx.kind, 0.01), None


def reference(p, x, depth, kind, norm, gate_act):
    bias = lambda name, i: p.get(f"{name}.{i}")
    r, y = x, _norm(x, norm, p["pre_weight.0"], bias("pre_bias", 0), 1e-5)
    for i in range(depth):
        z = _Linear.apply(y, p[f"fc1.{i}.weight"], p[f"fc1.{i}.bias"])
        h = _Linear.apply(_Act.apply(z, kind), p[f"fc2.{i}.weight"], p[f"fc2.{i}.bias"])
        u = _norm(h, norm, p[f"post_weight.{i}"], bias("post_bias", i), 1e-5) * p[f"scale.{i}"]
        if gate_act:
            u = u * getattr(torch, gate_act)(p[f"gate.{i}"])
        r = r + u
        y = _norm(r, norm, p[f"pre_weight.{i + 1}"], bias("pre_bias", i + 1), 1e-5)
    return y


def make(width, depth, seed, **kw):
    torch.manual_seed(seed)
    net = S.ResidualTrunk(width, depth, **kw)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n, p in net.named_parameters():
            if not n.startswith("fc"):
                p.add_(0.1 * torch.randn(p.shape, generator=g))
    return net


@pytest.mark.parametrize("rows,width,hidden,depth,kind,norm,gate,dtype,tol", [
    (130, 96, 200, 3, "gelu", "layer", "sigmoid", torch.float32, 4e-3),
    (77, 901, 130, 2, "silu", "rms", "tanh", torch.float32, 4e-3),
    (5, 40, None, 3, "leaky_relu", "layer", None, torch.float32, 4e-3),
    (300, 1300, 520, 2, "gelu", "rms", "sigmoid", torch.bfloat16, 6e-2),
    (64, 72, 264, 3, "silu", "layer", None, torch.bfloat16, 6e-2),
])
def test_trunk_against_64_bits(rows, width, hidden, depth, kind, norm, gate, dtype, tol):
    net = make(width, depth, 7, hidden=hidden, activation=kind, norm=norm, gate=gate, block_dtype=dtype)
    g = torch.Generator().manual_seed(11)
    x, up = torch.randn(rows, width, generator=g), torch.randn(rows, width, generator=g).to(dtype)
    p = {n: q.detach().double().requires_grad_() for n, q in net.named_parameters()}
    xr = x.double().requires_grad_()
    y = reference(p, xr, depth, kind, norm, gate)
    want = dict(zip(["x", *p], torch.autograd.grad(y, [xr, *p.values()], up.double())))
    net.cuda()
    xg = x.cuda().requires_grad_()
    out = net(xg)
    assert out.dtype == dtype and out.shape == x.shape
    out.backward(up.cuda())
    got = {"x": xg.grad, **{n: q.grad for n, q in net.named_parameters()}}
    for name, a, b in [("y", out.detach(), y.detach()), *((n, got[n], want[n]) for n in want)]:
        err = (a.double().cpu() - b).abs().max().item()
        assert err <= (2e-4 if name == "y" and dtype == torch.float32 else tol) * max(b.abs().max().item(), 1e-3), (name, err, b.abs().max().item())


def test_trunk_trains_with_the_fused_optimiser():
    """A step of FusedAdamW equals torch.optim.AdamW's on the same gradients (odd width: the norms' gradients are rows of one
    buffer), and two backward passes of equal networks agree bit for bit.  A parameter of at most 1.5 is rounded to 2^-24
    relative some four times (decay, step) and the step of at most lr = 1e-3 carries a few 2^-23: 5e-7 covers both."""
    x = torch.randn(200, 131, generator=torch.Generator().manual_seed(1)).cuda()
    nets = [make(131, 2, 3, gate="sigmoid").cuda() for _ in range(2)]
    opts = [S.FusedAdamW(nets[0].parameters(), lr=1e-3, weight_decay=0.01),
            torch.optim.AdamW(nets[1].parameters(), lr=1e-3, weight_decay=0.01)]
    for net in nets:
        net(x).square().mean().backward()
    for (n, a), b in zip(nets[0].named_parameters(), nets[1].parameters()):
        assert torch.equal(a.grad, b.grad), n
    for opt in opts:
        opt.step()
    for (n, a), b in zip(nets[0].named_parameters(), nets[1].parameters()):
        assert a.abs().max().item() <= 1.5 and (a - b).abs().max().item() <= 5e-7, n


def test_trunk_memory_per_block():
    """What a block keeps for its backward pass: its stream input in fp32, the block output in bf16, and checkpoints of three
    activations: 4 + 2 + (1 + 4 + 4) (1 + 1/64) bytes per stream element at hidden = 4 width; the gate, statistics and the
    allocator's rounding on top."""
    net = S.ResidualTrunk(512, 4, block_dtype=torch.bfloat16).cuda()
    x = torch.randn(4096, 512, device="cuda", requires_grad=True)
    net(x[:8]).sum().backward()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = net(x)
    torch.cuda.synchronize()
    kept = (torch.cuda.memory_allocated() - before) / (4 * 4096 * 512)
    assert kept <= (4 + 2 + 9 * (1 + 1 / 64)) * 1.02 + 2, kept      # + the last y


def test_trunk_without_gradients_is_the_same():
    net = make(200, 2, 5, gate="tanh", block_dtype=torch.bfloat16).cuda()
    x = torch.randn(3, 33, 200, device="cuda")
    with torch.no_grad():
        a = net(x)
    assert a.shape == x.shape and torch.equal(a, net(x))
