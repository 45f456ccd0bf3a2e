"""Refusals of the residual-trunk operators: decided on the host, before any launch, hence testable without a GPU."""
import ctypes as C

import pytest
import torch

from scpair_amd import _lib, ops

X, H = torch.zeros(4, 8), torch.zeros(4, 8)


@pytest.mark.parametrize("args,kw", [
    ((torch.zeros(()),), {}),
    ((X.half(),), {}),
    ((X.double(), H.double()), {}),
    ((X.bfloat16(), H), {}),                                         # a bf16 stream needs bf16 blocks
    ((X, torch.zeros(4, 7)), {}),
    ((X, torch.zeros(1, 8)), {}),
    ((X, H), {"pre": None}),
    ((X, H), {"pre": "batch"}),
    ((X, H), {"post": "batch"}),
    ((X, H), {"gate_act": "relu"}),
    ((X, H), {"eps": 0.0}),
    ((X, H), {"eps": float("nan")}),
    ((X, H), {"out_dtype": torch.bfloat16}),
    ((X, H), {"pre": "rms", "pre_bias": torch.zeros(8)}),
    ((X, H), {"post": "rms", "post_bias": torch.zeros(8)}),
    ((X, H), {"post_weight": torch.ones(8)}),
    ((X, H), {"pre_weight": torch.ones(7)}),
    ((X, H), {"pre_weight": torch.ones(8, dtype=torch.int32)}),
    ((X, H), {"scale": torch.ones(7)}),
    ((X, H), {"gate": torch.zeros(4)}),
    ((X, H), {"gate": torch.zeros(3, 8)}),
    ((X, H), {"gate": torch.zeros(4, 8, dtype=torch.bfloat16)}),     # a full gate has h's type
    ((X,), {"gate": X}),
    ((X,), {"scale": 0.5}),
    ((X,), {"post": "rms"}),
    ((X.bfloat16(),), {"out_dtype": torch.float32}),
    ((torch.zeros(2, 0), torch.zeros(2, 0)), {}),
    ((torch.zeros(1, 16385),), {}),
])
def test_gated_residual_norm_refuses(args, kw):
    with pytest.raises(ValueError):
        ops.gated_residual_norm(*args, **kw)


def test_gated_residual_norm_has_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.gated_residual_norm(X, H)


def test_residual_norm_c_entry_refuses():
    L = _lib.lib()
    assert L.scp_residual_norm_max_cols() == 16384

    def args(**kw):
        a = _lib.ResidualNorm()
        base = dict(x=64, h=64, r=64, y=64, stats=64, rows=2, cols=8, pre=1, ldx=8, ldh=8, eps=1e-5)
        for k, v in (base | kw).items():
            setattr(a, k, v)
        return C.byref(a)

    assert L.scp_residual_norm_fwd(None, None) == -1
    for bad in (dict(rows=0), dict(cols=0), dict(x=None), dict(ldx=-1), dict(pre=0), dict(pre=3), dict(post=3), dict(x_bf16=1),
                dict(gate_mode=4, gate=64), dict(gate_mode=1), dict(gate_act=3), dict(scale_mode=1), dict(y=None), dict(r=None),
                dict(h=None, post=1)):
        assert L.scp_residual_norm_fwd(args(**bad), None) == -1, bad
        assert L.scp_last_error()
    assert L.scp_residual_norm_fwd(args(cols=16385), None) == -2
    for bad in (dict(stats=None), dict(dw2=64), dict(dw1=64, ws=64), dict(dscale=64, ws=64), dict(dgate=64),
                dict(dy=64, lddy=-8)):
        assert L.scp_residual_norm_bwd(args(**bad), None) == -1, bad
    assert L.scp_residual_norm_bwd_ws_floats(0, 8) == 0
    assert L.scp_residual_norm_bwd_ws_floats(1, 900) == 5 * 900
