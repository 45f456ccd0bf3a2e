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
