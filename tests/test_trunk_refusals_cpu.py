"""More refusals of the residual-trunk operators and their C entries, decided on the host."""
import ctypes as C

import pytest
import torch

from scpair_amd import _lib, ops


def norm_args(**kw):
    a = _lib.ResidualNorm()
    for k, v in (dict(x=64, h=64, r=64, y=64, stats=64, rows=2, cols=8, pre=1, ldx=8, ldh=8, eps=1e-5) | kw).items():
        setattr(a, k, v)
    return C.byref(a)


@pytest.mark.parametrize("eps", [1e-50, 2.0 ** -150, 1e39, float("inf"), -1e-5])
def test_eps_that_fp32_cannot_hold(eps):
    """0 or infinity in fp32: a row of zeros would have no norm, or no row one."""
    with pytest.raises(ValueError, match="eps"):
        ops.gated_residual_norm(torch.zeros(4, 8), eps=eps)
    L = _lib.lib()
    f = C.c_float(eps).value
    assert L.scp_residual_norm_fwd(norm_args(eps=f), None) == -1 and b"eps" in L.scp_last_error()
    assert L.scp_residual_norm_bwd(norm_args(eps=f), None) == -1 and b"eps" in L.scp_last_error()


@pytest.mark.parametrize("bad", [dict(b1=64), dict(w1=64), dict(scale_mode=1, scale=64), dict(scale_mode=2, scale=64)])
def test_parts_of_a_block_without_one(bad):
    """h null: the backward pass took b1 into its recomputed row, and gradients of the others stayed unwritten."""
    L = _lib.lib()
    for entry in (L.scp_residual_norm_fwd, L.scp_residual_norm_bwd):
        assert entry(norm_args(h=None, **bad), None) == -1 and b"without a block" in L.scp_last_error()


def test_gradients_of_an_absent_block():
    L = _lib.lib()
    assert L.scp_residual_norm_bwd(norm_args(h=None, dh=64, dx=64), None) == -1 and b"absent" in L.scp_last_error()


@pytest.mark.parametrize("M,N,K", [(4096, 4096, 4096), (16384, 4096, 4096)])
def test_workspace_of_the_fp32_blocks(M, N, K):
    """What the documentation says of the wide products in the fp32-equivalent precision: 12 bytes an element of x and W forward, of dy and W
    backward, and three fp32 planes of dW."""
    a = _lib.Linear8()
    for k, v in dict(x=4096, W=4096, y=4096, dy=4096, dx=4096, dW=4096, codes=4096, steps=4096, M=M, N=N, K=K, ldx=K, lddy=N, ns=3).items():
        setattr(a, k, v)
    tiles, L = (C.c_int * 3)(), _lib.lib()
    assert L.scp_linear8_tiles(C.byref(a), tiles) == 0 and list(tiles) == [256] * 3
    assert L.scp_linear8_fwd_ws(C.byref(a)) == 12 * (M * K + N * K)
    bwd = L.scp_linear8_bwd_ws(C.byref(a))
    assert 0 <= bwd - (12 * (M * N + N * K) + 12 * N * K) <= 8 * N * K          # and slabs where a sum is divided
    assert L.scp_linear8_tiles(None, tiles) == -1 and L.scp_linear8_tiles(C.byref(a), None) == -1
