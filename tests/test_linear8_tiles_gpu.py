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
