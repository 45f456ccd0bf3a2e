"""gelu (bf16) and silu of ops.act8 far left of zero, where the values are small but not zero: relative accuracy.

Tolerances, relative to the value.  bf16: half a step, 2^-8, and 2^-12 for the evaluation (normal distribution function to 1.4e-5, the
exponential of an argument of up to 72 with fp32's rounding of that argument, 72 * 3 * 2^-24 = 1.3e-5).  fp32 silu: exp(-x) with the
rounding of its argument, (32 + 4 |x|) * 2^-24.  (fp32 gelu is 1 + erf, whose error is absolute: test_ckpt8_gpu.py.)  The
distribution function in 64 bits is taken from erfc: torch.special.ndtr is 0 below -8.3."""
import math

import pytest
import torch

from tests.test_ckpt8_gpu import B16, E, F32, act_ref, act_slope_ref, pack_ref

pytestmark = pytest.mark.gpu


def grid(lo, hi, dtype):
    if dtype == B16:      # every value
        bits = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16)
        x = bits.view(B16)
        return x[(x >= lo) & (x <= hi)]
    return torch.linspace(lo, hi, 20001)


def slack(x, dtype):
    return 2.0 ** -8 + 2.0 ** -12 if dtype == B16 else (32 + 4 * x.double().abs()) * E


def reference(x, kind):
    """value and derivative"""
    if kind == "silu":
        return act_ref(x, kind, 0.0), act_slope_ref(x, kind, 0.0)
    cdf = 0.5 * torch.erfc(-x * math.sqrt(0.5))
    return x * cdf, cdf + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("kind,dtype", [("gelu", B16), ("silu", B16), ("silu", F32)])
def test_values_and_derivatives_left_of_zero(kind, dtype):
    from scpair_amd import ops
    x = grid(-12.0, -3.0, dtype)
    z = torch.zeros(x.numel(), 64, dtype=dtype)          # one value to a group
    z[:, 0] = x
    zg = z.cuda().requires_grad_()
    a = ops.act8(zg, kind)
    want = reference(x.double(), kind)[0]
    assert (want < 0).all() and ((a.detach()[:, 0].cpu().double() - want).abs() <= slack(x, dtype) * want.abs()).all()
    d, = torch.autograd.grad(a, zg, torch.ones_like(z).cuda())
    v = pack_ref(z)[2][:, 0]
    want = reference(v, kind)[1]
    assert (want < 0).all() and ((d[:, 0].cpu().double() - want).abs() <= slack(v, dtype) * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, B16])
def test_gelu_everywhere_else(dtype):
    """From -3 up: the distribution function to 2^-22 absolute (fit 1.9e-7, fp32 evaluation a few 2^-24), times x; half a step.
    Below 2^-126 the steps of bf16 no longer shrink with the value: they are 2^-133, half a step 2^-134."""
    from scpair_amd import ops
    x = grid(-3.0, 40.0, dtype).reshape(1, -1)
    want = act_ref(x.double(), "gelu", 0.0)
    got = ops.act8(x.cuda(), "gelu").cpu().double()
    assert ((got - want).abs() <= x.double().abs() * 2.0 ** -21 + want.abs() * (2.0 ** -8 if dtype == B16 else E) + 2.0 ** -134).all()


def test_silu_of_every_bf16_is_the_nearest_bf16():
    """From -87 up (exp(x) below it is no normal fp32 number), magnitudes from 2^-120 up (values are normal bf16 numbers)."""
    from scpair_amd import ops
    x = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(B16)
    x = x[torch.isfinite(x) & (x >= -87) & (x.abs() >= 2.0 ** -120)]
    want = act_ref(x.double(), "silu", 0.0).to(B16)
    assert x.numel() > 40000 and torch.equal(ops.act8(x.reshape(1, -1).cuda(), "silu").cpu()[0], want)


@pytest.mark.parametrize("kind,slope", [("leaky_relu", 0.0), ("leaky_relu", 0.1), ("gelu", 0.0), ("silu", 0.0)])
@pytest.mark.parametrize("dtype", [F32, B16])
def test_a_group_without_values_has_no_derivatives(kind, slope, dtype):
    """A group that held an infinity or a NaN reads as NaN, and so does the gradient of all its columns, for every activation: the sign
    that a leaky relu would need is not there."""
    from scpair_amd import ops
    z = torch.randn(3, 130, generator=torch.Generator().manual_seed(2)).to(dtype)
    z[0, 70], z[2, 129] = float("inf"), float("nan")
    zg = z.cuda().requires_grad_()
    d, = torch.autograd.grad(ops.act8(zg, kind, slope), zg, torch.ones(3, 130, dtype=dtype).cuda())
    bad = torch.zeros(3, 130, dtype=torch.bool)
    bad[0, 64:128], bad[2, 128:] = True, True
    assert torch.equal(d.cpu().isnan(), bad)
