"""HipLinear8 in the place of HipLinear: the same arguments, and the same output and input and bias gradient up to the kernels' rounding
(fp32-equivalent products: 2^-22 per term pair on top of K / 16 + 16 steps of 2^-24, twice, for the two kernels compared)."""
import pytest
import torch

import scpair_amd as S
from tests.test_ckpt8_gpu import E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("relu", [False, True])
def test_stands_in_for_its_base(relu):
    torch.manual_seed(4)
    a = S.HipLinear(130, 70).cuda()
    b = S.HipLinear8(130, 70).cuda()
    b.load_state_dict(a.state_dict())
    x, up = torch.randn(90, 130).cuda(), torch.randn(90, 70).cuda()
    runs = []
    for net in (a, b):
        xl = x.clone().requires_grad_()
        y = net(xl, relu_input=relu)
        runs.append([y.detach(), *torch.autograd.grad(y, (xl, net.bias), up)])
    xin = x.relu() if relu else x
    terms = [xin.abs() @ a.weight.abs().t() + a.bias.abs(), up.abs() @ a.weight.abs(), up.abs().sum(0)]
    for p, q, t in zip(*runs, terms):
        assert ((p - q).abs() <= 2 * (6 * 130 / 16 + 16 + 4) * E * t).all()
    if relu:
        assert not runs[1][1][x < 0].any()
